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
  const void* zero = nullptr;                                        // 16 bytes of zeros: where the loads of absent rows point
};
// the launch that seq_plan() chose for these sizes: rows per workgroup, whether the waves share the keys (false: each takes keys of its own)
struct SeqPlan { int shared = 1, rows = 128, splits = 1, chunk = 0; };
SeqPlan seq_plan(const SeqArgs& a, int compute_units);
hipError_t launch_seq_fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s);
hipError_t launch_seq_join(const SeqArgs& a, hipStream_t s);

struct SeqGradArgs {
  SeqArgs f;
  const void* dout = nullptr; long long lddo = 0;
  void *dq = nullptr, *dk = nullptr, *dv = nullptr; long long lddq = 0, lddk = 0, lddv = 0;
  float* delta = nullptr;                                            // [heads][rows_q] scratch: sum_d dout * out of every row
};
hipError_t launch_seq_grad(const SeqGradArgs& a, hipStream_t s);

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

// Tiles in LDS: rows of DP elements, 16-byte chunks; chunk c of row r lies at c ^ (r & 7), so that the 32 rows that one matrix operand reads
// at the same chunk spread over the banks (a row is 128, 256 or 512 bytes: without it they share eight lanes' worth of banks).
template <typename T, int DP> struct SeqTile {
  static constexpr int kRow = DP * (int)sizeof(T);           // bytes
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPer = 16 / (int)sizeof(T);           // elements of a chunk
  static __device__ __forceinline__ int at(int r, int c) { return r * kRow + ((c ^ (r & 7)) << 4); }
};
// operand with rows along the lanes: elements 8 u .. 8 u + 7 of row r
template <typename T, int DP>
__device__ __forceinline__ typename SeqVec<T>::v8 seq_row(const char* tile, int r, int u) {
  typedef SeqTile<T, DP> L;
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const typename SeqVec<T>::v8*>(tile + L::at(r, u));
  } else {
    const sq_f4 a = *reinterpret_cast<const sq_f4*>(tile + L::at(r, 2 * u)), b = *reinterpret_cast<const sq_f4*>(tile + L::at(r, 2 * u + 1));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
// operand with columns along the lanes: column 32 cb + (lane & 31), k-slot (g, e) = row r0 + (e & 3) + 4 g + 8 (e >> 2) -- the order in which
// a product's registers 8 t .. 8 t + 7 hold its rows, so the other operand of the next product comes straight out of them.  16 bits: two
// transposing LDS reads (a 16-lane group reads a 4 x 16 block, lane i gets column i).
template <typename T, int DP>
__device__ __forceinline__ typename SeqVec<T>::v8 seq_col(const char* tile, int r0, int cb, int lane) {
  typedef SeqTile<T, DP> L;
  const int g = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int i = lane & 15, r = r0 + 4 * g + (i >> 2), c = cb * 4 + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
    typedef __attribute__((address_space(3))) sq_s4* lp;
    const sq_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(tile + L::at(r, c) + (i & 1) * 8));
    const sq_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(tile + L::at(r + 8, c) + (i & 1) * 8));
    return __builtin_bit_cast(typename SeqVec<T>::v8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    sq_f8 v;
    const int d = 32 * cb + (lane & 31);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = r0 + 4 * g + (e & 3) + 8 * (e >> 2);
      v[e] = *reinterpret_cast<const float*>(tile + L::at(r, d >> 2) + (d & 3) * 4);
    }
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
// sixteen bytes (or thirty-two in 32 bits) of a row in memory: elements 8 u .. 8 u + 7, zeros where `ok` is false
template <typename T> __device__ __forceinline__ typename SeqVec<T>::v8 seq_load8(const T* p, bool ok) {
  typename SeqVec<T>::v8 v = {};
  if (ok) v = *reinterpret_cast<const typename SeqVec<T>::v8*>(p);
  return v;
}
template <typename T> __device__ __forceinline__ void seq_store4(T* p, float a, float b, float c, float d) {
  const sq_f4 v = {a, b, c, d};
  if constexpr (sizeof(T) == 4) *reinterpret_cast<sq_f4*>(p) = v;
  else *reinterpret_cast<typename SeqVec<T>::v4*>(p) = __builtin_convertvector(v, typename SeqVec<T>::v4);
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
// 16 bytes from memory straight to LDS: lane i's sixteen bytes land at dst + 16 i
__device__ __forceinline__ void seq_dma16(const void* src, char* dst) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// The sequence and the tile in it that a workgroup's tile index names: every sequence of n rows has ceil(n * mult / rows) tiles.  Starts that
// run backwards or leave the tensor are clamped: such a sequence is empty, nothing outside the tensor is touched.
struct SeqWhere { int b, tile, start, n; };
__device__ __forceinline__ bool seq_find(const int32_t* cu, int batch, int total, int mult, int rows, int index, SeqWhere& w) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    const int b = b0 + lane;
    int s = 0, e = 0;
    if (b < batch) { s = cu[b]; e = cu[b + 1]; }
    s = s < 0 ? 0 : (s > total ? total : s);
    e = e < s ? s : (e > total ? total : e);
    const int n = e - s;
    const int t = (int)(((long long)n * mult + rows - 1) / rows);
    int x = t;                                             // inclusive scan over the 64 sequences
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int y = __shfl_up(x, o, 64); if (lane >= o) x += y; }
    const unsigned long long m = __builtin_amdgcn_ballot_w64(index < before + x);
    if (m) {
      const int src = __builtin_ctzll(m);
      w.b = b0 + src;
      w.tile = index - before - __shfl(x - t, src, 64);
      w.start = __shfl(s, src, 64);
      w.n = __shfl(n, src, 64);
      w.b = __builtin_amdgcn_readfirstlane(w.b); w.tile = __builtin_amdgcn_readfirstlane(w.tile);
      w.start = __builtin_amdgcn_readfirstlane(w.start); w.n = __builtin_amdgcn_readfirstlane(w.n);
      return true;
    }
    before += __shfl(x, 63, 64);
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
