// Operators on packed sequences and on the paged key / value cache: what the host hands to their kernels, and the device pieces that the
// forward (sequence_fwd.hip), backward (sequence_bwd.hip) and cache (sequence_cache.hip) kernels share.
#pragma once
#include "common.h"

namespace vnr {

enum { SEQ_F32 = 0, SEQ_F16 = 1, SEQ_BF16 = 2 };

struct SeqArgs {
  int dtype = 0, batch = 0, heads = 0, kv_heads = 0, dim = 0, causal = 0;
  float scale = 1.f;
  int rows_q = 0, rows_k = 0;
  const int32_t* cu_q = nullptr; const int32_t* cu_k = nullptr;      // [batch + 1] first rows of the sequences
  const void *q = nullptr, *k = nullptr, *v = nullptr;               // packed rows; paged: k, v = the pools [pages][kv_heads][page_size][dim]
  long long ldq = 0, ldk = 0, ldv = 0, ldo = 0;                      // elements from one row to the next
  void* out = nullptr; float* lse = nullptr;                         // lse [heads][rows_q], natural logarithm
  // paged
  const int32_t* ctx = nullptr; const int32_t* table = nullptr;      // [batch] keys in front of the new ones, [batch][table_width] pages
  int table_width = 0, page_shift = 0, pages = 0, max_context = 0, max_new = 0;
  // a sequence's keys cut into `splits` pieces of `chunk` keys, joined by seq_join_kernel; part [splits][rows_q * heads][dim], ml [splits][rows_q * heads][2]
  int splits = 1, chunk = 0;
  float* part = nullptr; float* ml = nullptr;
  const void* zero = nullptr;                                        // 64 bytes of zeros: where the loads of absent rows point
};
// the launch that seq_plan() chose for these sizes: how many of a workgroup's four waves stand side by side along the rows (the others: along the keys)
struct SeqPlan { int row_waves = 4, splits = 1, chunk = 0; };
SeqPlan seq_plan(const SeqArgs& a, int compute_units);
bool seq_fwd_fits(const SeqArgs& a, const SeqPlan& p);       // do the grids hold that many rows and heads? (a launch has at most 2^32 - 1 threads)
bool seq_grad_fits(const SeqArgs& a);
hipError_t launch_seq_fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s);
hipError_t launch_seq_join(const SeqArgs& a, hipStream_t s);

struct SeqGradArgs {
  SeqArgs f;
  const void* dout = nullptr; long long lddo = 0;
  void *dq = nullptr, *dk = nullptr, *dv = nullptr; long long lddq = 0, lddk = 0, lddv = 0;
  float* delta = nullptr;                                            // [2][heads][rows_q] scratch: sum_d dout * out of every row; its lse in units of log2, less the lift of the weights
};
hipError_t launch_seq_grad(const SeqGradArgs& a, int compute_units, hipStream_t s);

struct SeqAppendArgs {
  int dtype = 0, batch = 0, heads = 0, kv_heads = 0, dim = 0, rows = 0;
  const int32_t* cu = nullptr; const int32_t* ctx = nullptr; const int32_t* table = nullptr;
  int table_width = 0, page_shift = 0, pages = 0;
  const void *k = nullptr, *v = nullptr, *q = nullptr; long long ldk = 0, ldv = 0, ldq = 0, ldqo = 0;
  void *kc = nullptr, *vc = nullptr, *q_out = nullptr;
  const float* rotation = nullptr; int rot_dim = 0, interleaved = 0;
};
hipError_t launch_seq_append(const SeqAppendArgs& a, hipStream_t s);
hipError_t launch_rotation_table(int positions, int rot_dim, double base, float* out, hipStream_t s);

#if defined(__HIPCC__)
typedef float sq_f2 __attribute__((ext_vector_type(2)));
typedef float sq_f4 __attribute__((ext_vector_type(4)));
typedef float sq_f8 __attribute__((ext_vector_type(8)));
typedef short sq_s4 __attribute__((ext_vector_type(4)));
typedef __bf16 sq_bf16;
template <typename T> struct SeqVec;                       // eight / four / two elements of a type
template <> struct SeqVec<sq_bf16> { typedef __bf16 v8 __attribute__((ext_vector_type(8))); typedef __bf16 v4 __attribute__((ext_vector_type(4))); };
template <> struct SeqVec<_Float16> { typedef _Float16 v8 __attribute__((ext_vector_type(8))); typedef _Float16 v4 __attribute__((ext_vector_type(4))); };
template <> struct SeqVec<float> { typedef sq_f8 v8; typedef sq_f4 v4; };

// D += A . B over 16 k: lane (r = lane & 31, g = lane >> 5) holds k-slots 8 g .. 8 g + 7 of row r of A / column r of B; D: column r, rows
// 8 (i / 4) + 4 g + (i % 4) in register i.  In 32 bits the sixteen slots go through eight 32x32x2 products (a slot pair (e, 8 + e) each).
__device__ __forceinline__ f32x16 seq_mma(SeqVec<sq_bf16>::v8 a, SeqVec<sq_bf16>::v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 seq_mma(SeqVec<_Float16>::v8 a, SeqVec<_Float16>::v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 seq_mma(sq_f8 a, sq_f8 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// Tiles in LDS: rows of DP elements in 16-byte chunks; chunk c of row r lies at c ^ turn(r).  Two kinds of reads have to spread over the 64
// banks (256 bytes): sixteen rows at one chunk (the phases of a 16-byte read take rows 0-3, 12-15, 20-27 together), and four consecutive rows
// at four neighbouring chunks (half a wave of the transposing read).  With turn(r) = r % 8 the second kind met 4-fold conflicts: 62 % of the
// LDS cycles of the backward kernels.
template <typename T, int DP> struct SeqTile {
  static constexpr int kRow = DP * (int)sizeof(T);           // bytes
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPer = 16 / (int)sizeof(T);           // elements of a chunk
  static __device__ __forceinline__ int turn(int r) {        // rows of 128 bytes: two of them share the banks
    return kChunks == 8 ? ((r & 2) << 1) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * kRow + ((c ^ turn(r)) << 4); }
};
// Where a lane reads its operands in a tile (bytes of LDS).  row: lane (r = lane & 31, g = lane >> 5) reads elements 16 t + 8 g .. + 7 of row r;
// col: column 32 cb + r, k-slot (g, e) = row r0 + (e & 3) + 4 g + 8 (e >> 2) -- the order in which a product's registers 8 t .. 8 t + 7 hold
// its rows, so the other operand of the next product comes straight out of them.  Everything that varies inside a tile is an exclusive or of
// the address with a constant (turn() again), so two registers do for all of a tile's reads -- as long as the compiler does not keep every one
// of the addresses: seq_at() hides the sum of tile and lane from it, once a tile.
template <typename T, int DP> struct SeqReads {
  typedef SeqTile<T, DP> L;
  unsigned row, col;
  __device__ __forceinline__ void set(int lane) {
    const int r = lane & 31, g = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, q = 4 * g + (i >> 2);         // transposing reads: a 16-lane group reads a 4 x 16 block, lane i gets column i
      row = L::at(r, g);
      col = L::at(q, ((lane >> 4) & 1) * 2 + ((i & 3) >> 1)) + (i & 1) * 8;
    } else {
      row = L::at(r, 2 * g);
      col = L::at(4 * g, r >> 2) + (r & 3) * 4;
    }
  }
};
__device__ __forceinline__ unsigned seq_at(unsigned tile, unsigned lane) {
  unsigned x = tile + lane;
  asm volatile("" : "+v"(x));
  return x;
}
template <typename V> __device__ __forceinline__ V seq_ds(unsigned at) { return *(const __attribute__((address_space(3))) V*)at; }
// A run of N products whose operands come from LDS, two at a time: the next two reads are issued in front of these two products.  Left alone the
// compiler saves registers it need not save -- read, wait for LDS, multiply, read ... -- and every product waits out a read: 4 prompts of up to 4096
// rows (32 heads of 128, bf16) 435 us so, 417 us here; four at a time 421.  (0x406: arithmetic and scalar work may still cross.)
template <typename T, int N, typename Load, typename Mul> __device__ __forceinline__ void seq_run(Load&& load, Mul&& mul) {
  constexpr int B = 2;
  static_assert(N % B == 0, "whole batches");
  typename SeqVec<T>::v8 x[2][B];
#pragma unroll
  for (int i = 0; i < B; ++i) x[0][i] = load(i);
#pragma unroll
  for (int b = 0; b < N / B; ++b) {
    if (b + 1 < N / B) {
#pragma unroll
      for (int i = 0; i < B; ++i) x[(b + 1) & 1][i] = load((b + 1) * B + i);
    }
    __builtin_amdgcn_sched_barrier(0x406);
#pragma unroll
    for (int i = 0; i < B; ++i) mul(b * B + i, x[b & 1][i]);
    __builtin_amdgcn_sched_barrier(0x406);
  }
}
// at: seq_at(tile, reads.row); rows r0 .. r0 + 31 of the tile
template <typename T, int DP> __device__ __forceinline__ typename SeqVec<T>::v8 seq_row(unsigned at, int r0, int t) {
  typedef SeqTile<T, DP> L;
  if constexpr (sizeof(T) == 2) {
    return seq_ds<typename SeqVec<T>::v8>((at ^ (t << 5)) + r0 * L::kRow);
  } else {
    const sq_f4 a = seq_ds<sq_f4>((at ^ (t << 6)) + r0 * L::kRow), b = seq_ds<sq_f4>((at ^ (t << 6) ^ 16) + r0 * L::kRow);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
// at: seq_at(tile, reads.col); r0: a multiple of 16
template <typename T, int DP> __device__ __forceinline__ typename SeqVec<T>::v8 seq_col(unsigned at, int r0, int cb) {
  typedef SeqTile<T, DP> L;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) sq_s4* lp;
    const sq_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)((at ^ (cb << 6)) + r0 * L::kRow));
    const sq_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)((at ^ (cb << 6) ^ 32) + (r0 + 8) * L::kRow));
    return __builtin_bit_cast(typename SeqVec<T>::v8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    sq_f8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = seq_ds<float>((at ^ (cb << 7) ^ ((e & 3) << 6) ^ ((e >> 2) << 5)) + (r0 + (e & 3) + 8 * (e >> 2)) * L::kRow);
    return v;
  }
}
// eight accumulator registers 8 t .. 8 t + 7 as an operand, rounded once to the type
template <typename T> __device__ __forceinline__ typename SeqVec<T>::v8 seq_pack(const f32x16& x, int t) {
  sq_f8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[8 * t + e];
  if constexpr (sizeof(T) == 4) return v; else return __builtin_convertvector(v, typename SeqVec<T>::v8);
}
// the same with what the rounding left, rounded in turn: twice the bits for one product more
template <typename T> __device__ __forceinline__ typename SeqVec<T>::v8 seq_pack(const f32x16& x, int t, typename SeqVec<T>::v8& rest) {
  static_assert(sizeof(T) == 2, "32 bits leave nothing");
  sq_f8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[8 * t + e];
  typename SeqVec<T>::v8 r = __builtin_convertvector(v, typename SeqVec<T>::v8);
  sq_f4 bits = __builtin_bit_cast(sq_f4, r);
  asm("" : "+v"(bits));                                      // one rounding for both uses
  r = __builtin_bit_cast(typename SeqVec<T>::v8, bits);
  rest = __builtin_convertvector(v - __builtin_convertvector(r, sq_f8), typename SeqVec<T>::v8);
  return r;
}
// Values that are not finite in a tile whose keys some row does not see: 0 times them would reach that row.  seq_tainted: does the tile hold any
// (threads first, first + step, ... take its 16-byte chunks)?
template <typename T, int DP, int ROWS> __device__ __forceinline__ bool seq_tainted(const char* tile, int first, int step) {
  unsigned top = 0;
  for (int q = first; q < ROWS * SeqTile<T, DP>::kChunks; q += step) {
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    const u4 x = *reinterpret_cast<const u4*>(tile + q * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned hi = sizeof(T) == 4 ? x[e] & 0x7fffffffu : x[e] & 0x7fff0000u, lo = sizeof(T) == 4 ? 0u : (x[e] << 16) & 0x7fff0000u;
      top = top > hi ? top : hi; top = top > lo ? top : lo;
    }
  }
  const unsigned limit = __is_same(T, _Float16) ? 0x7c000000u : 0x7f800000u;
  return __builtin_amdgcn_ballot_w64(top >= limit) != 0;
}
// They become zeros in the tile, and what[0 / 1 / 2][channel] the first key (k0: the tile's first) with plus infinity / minus infinity / no number
// there: a row sees a prefix of the keys, so it sees one of them if and only if it sees the first.
template <typename T, int DP, int ROWS> __device__ __forceinline__ void seq_apart(char* tile, int* what, int k0, int first, int step) {
  typedef SeqTile<T, DP> L;
  for (int q = first; q < ROWS * L::kChunks; q += step) {
    const int r = q / L::kChunks, c = (q % L::kChunks) ^ L::turn(r);
    T* x = reinterpret_cast<T*>(tile + q * 16);
    for (int e = 0; e < L::kPer; ++e) {
      const float v = (float)x[e];
      if (__builtin_fabsf(v) < __builtin_inff()) continue;
      atomicMin(what + (v != v ? 2 : v > 0.f ? 0 : 1) * DP + c * L::kPer + e, k0 + r);
      x[e] = (T)0.f;
    }
  }
}

// elements 8 u .. 8 u + 7 of a row in memory, zeros where `ok` is false (read from `zero`: no branch)
template <typename T> __device__ __forceinline__ typename SeqVec<T>::v8 seq_load8(const T* p, bool ok, const void* zero) {
  return *reinterpret_cast<const typename SeqVec<T>::v8*>(ok ? (const void*)p : zero);
}
template <typename T> __device__ __forceinline__ void seq_store4(T* p, float a, float b, float c, float d) {
  const sq_f4 v = {a, b, c, d};
  if constexpr (sizeof(T) == 4) *reinterpret_cast<sq_f4*>(p) = v;
  else *reinterpret_cast<typename SeqVec<T>::v4*>(p) = __builtin_convertvector(v, typename SeqVec<T>::v4);
}
// operands that a loop keeps reading are waited for here, not by a counter wait that the compiler would repeat in every turn of the loop (and
// that would drain the transfers on their way)
template <typename V, int N> __device__ __forceinline__ void seq_settle(V (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const sq_f4* p = reinterpret_cast<const sq_f4*>(&x[i]);
#pragma unroll
    for (int j = 0; j < (int)(sizeof(V) / 16); ++j) asm volatile("" ::"v"(p[j]));
  }
}
// the value of the lane itself and of the one 32 away, in either order
__device__ __forceinline__ sq_f2 seq_pair(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const sq_f2 v = {__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])};
  return v;
}
__device__ __forceinline__ float seq_pair_max(float x) { const sq_f2 v = seq_pair(x); return fmaxf(v[0], v[1]); }
__device__ __forceinline__ float seq_pair_sum(float x) { const sq_f2 v = seq_pair(x); return v[0] + v[1]; }
// 16 (4) bytes a lane from memory straight to LDS: lane i's land at dst + 16 i (4 i); dst is the same for the wave.  The compiler is not told
// of the transfer -- it would drain all of them in front of every transposing read of LDS --: seq_dma_wait in front of the barrier behind
// which the tile is read is the kernels' own duty.  (No register is written, and the counter waits that the compiler places for its own loads
// only become longer by transfers it does not know.  m0, the transfer's destination, is set and used inside the block; nothing else in these
// kernels uses it.)
__device__ __forceinline__ unsigned seq_lds(const char* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) char*)p; }
__device__ __forceinline__ void seq_dma16(const void* src, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
}
// the same from a scalar base and a 32-bit offset a lane: no address arithmetic in vector registers
__device__ __forceinline__ void seq_dma16(const void* base, unsigned offset, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void seq_dma4(const void* src, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(src) : "memory");
}
// the wave's transfers have landed
__device__ __forceinline__ void seq_dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The offsets of a wave's lanes in its transfers of 64 chunks (kRowsOf rows, `ld` bytes apart, ld a multiple of a tile's row): turn() of a sum of
// rows without common bits is the exclusive or of their turns, and what a transfer's first row adds stays inside the row.  One register.
template <typename T, int DP> struct SeqLanes {
  typedef SeqTile<T, DP> L;
  static constexpr int kRowsOf = 64 / L::kChunks;
  unsigned base;
  __device__ __forceinline__ void set(unsigned ld, int lane, int first) {      // first: the wave's first transfer of a tile, a power of two's multiple of its count
    const int r = lane / L::kChunks;
    base = r * ld + (((lane % L::kChunks) ^ L::turn(r) ^ L::turn(first * kRowsOf)) << 4);
  }
  __device__ __forceinline__ unsigned at(int i) const { return base ^ (unsigned)(L::turn(i * kRowsOf) << 4); }       // of the wave's i-th
};
// a load through the scalar cache: `p` is the same for the wave and nobody writes there during the kernel
__device__ __forceinline__ int seq_scalar(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int*)(unsigned long long)p;
}

// A sequence's rows, by one rule for every operator: its starts are clamped to the tensor, and one whose end lies in front of its start is empty
__device__ __forceinline__ void seq_clamp(int s, int e, int total, int& start, int& n) {
  s = s < 0 ? 0 : (s > total ? total : s);
  e = e < s ? s : (e > total ? total : e);
  start = s; n = e - s;
}
// The sequence that owns row `token` (the first where starts overlap; -1: none) and its first row: 64 sequences a look
__device__ __forceinline__ int seq_owner(const int32_t* cu, int batch, int total, int token, int& start) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    int s = 0, n = 0;
    if (b0 + lane < batch) seq_clamp(cu[b0 + lane], cu[b0 + lane + 1], total, s, n);
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(s <= token && token < s + n);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      start = __builtin_amdgcn_readlane(s, src);
      return b0 + src;
    }
  }
  return -1;
}
// The sequence and the tile in it that a workgroup's tile index names: every sequence of n rows has ceil(n * mult / rows) tiles.  Nothing
// outside the tensor is touched, whatever the starts are.  `other` (or null): x0 =
// other[b], x1 = other[b + two], fetched along with the starts.  Where the launch has more workgroups than the chip
// holds at once, up to 64 sequences are gone through from the longest (rows, or rows + x0 where x0 counts keys in front of them: `two` 0) to
// the shortest: it ends with its short tasks (eight chunks of up to 512 rows over up to 6000 keys: 223 -> 187 us; about 1 us of a small launch).
struct SeqWhere { int b, rank, tile, start, n, x0, x1; };         // rank: of the sequence in the order of the tasks
__device__ __forceinline__ bool seq_find(const int32_t* cu, int batch, int total, int mult, int rows, int index, const int32_t* other, int two, SeqWhere& w) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    int b = b0 + lane;
    int s = 0, e = 0, x0 = 0, x1 = 0;
    if (b < batch) {
      s = cu[b]; e = cu[b + 1];
      if (other) { x0 = other[b]; x1 = other[b + two]; }
    }
    int n;
    seq_clamp(s, e, total, s, n);
    int t = (int)(((long long)n * mult + rows - 1) / rows);
    if (gridDim.x > 512 && batch > 1 && batch <= 64) {       // ranks, then everything to the lane of its rank
      const int key = b < batch ? n + (two ? 0 : x0 < 1 << 30 ? x0 : 1 << 30) : -1;
      int rank = 0;
      for (int j = 0; j < batch; ++j) { const int k = __builtin_amdgcn_readlane(key, j); rank += (k > key || (k == key && j < lane)) ? 1 : 0; }
      rank = b < batch ? rank : lane;
      auto to = [&](int v) { return __builtin_amdgcn_ds_permute(rank << 2, v); };
      b = to(b); s = to(s); n = to(n); t = to(t); x0 = to(x0); x1 = to(x1);
    }
    int x = t;                                               // inclusive scan over the 64 sequences
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int y = __shfl_up(x, o, 64); if (lane >= o) x += y; }
    const unsigned long long m = __builtin_amdgcn_ballot_w64(index < before + x);
    if (m) {
      const int src = __builtin_ctzll(m);
      w.rank = b0 + src;
      w.tile = index - before - __builtin_amdgcn_readlane(x - t, src);
      w.b = __builtin_amdgcn_readlane(b, src); w.start = __builtin_amdgcn_readlane(s, src); w.n = __builtin_amdgcn_readlane(n, src);
      w.x0 = __builtin_amdgcn_readlane(x0, src); w.x1 = __builtin_amdgcn_readlane(x1, src);
      return true;
    }
    before += __builtin_amdgcn_readlane(x, 63);
  }
  return false;
}
// workgroup -> task: the hardware deals workgroups to the 8 XCDs in turn, the tasks of one XCD are to be neighbours (the same keys in its L2)
__device__ __forceinline__ int seq_task(int id, int n) {
  const int per = n >> 3, rest = n & 7, x = id & 7, i = id >> 3;
  return x * per + (x < rest ? x : rest) + i;
}
#endif
}  // namespace vnr
