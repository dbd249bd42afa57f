// Attention forward on packed sequences and over a paged cache: out = softmax(scale q k' + mask) v, one pass over the keys with the running
// maximum and sum of every row.
//
//   S' = K Q'   (keys along the product's rows, the 32 query rows of a tile along its columns: a lane owns ONE query row, its maximum and
//               sum are register arithmetic plus one exchange with the lane 32 away)
//   P  = exp2(c S - c m), c = scale log2 e; m is a running bound of the row: it moves only when a tile exceeds it by more than 8 / c, so that
//        the accumulators are rarely rescaled.  P is rounded to the operands' type (relative 2^-9 / 2^-12, nothing in 32 bits) for the second
//        product; the row sums take the unrounded values, in 32 bits
//   O' += V' P'  with P' straight out of the first product's registers (sequence.h: seq_col's key order)
//
// K and V tiles come straight from memory to LDS (16 bytes a lane, no registers), the next tile while this one is multiplied.
#include "sequence.h"

namespace vnr {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kBound = 8.f;                                // how far (log2) a row may exceed its running bound before it is moved
constexpr int kMaxSplits = 64;

// Where the rows of a task's keys and values are, 16 bytes at a time.  `n`: keys of the sequence; rows from n on read as zeros.
template <typename T, int DP, bool PAGED>
struct KeySource {
  typedef SeqTile<T, DP> L;
  static constexpr int kRowsOf = 64 / (L::kChunks < 64 ? L::kChunks : 64);       // rows of one 64-lane transfer (a row is at most 512 bytes)
  const T *k, *v; long long ldk, ldv; const int32_t* table; int shift, pages, kv_heads, head, dim, n; const void* zero;
  __device__ __forceinline__ int page_of(int row) const { return row < n ? table[row >> shift] : -1; }
  // transfer `i` of a tile that starts at key k0; page: the row's page (PAGED)
  __device__ __forceinline__ void to_lds(int k0, int i, int page, char* tk, char* tv, int lane) const {
    const int r = i * kRowsOf + lane / L::kChunks, c = (lane % L::kChunks) ^ (r & 7);
    const int row = k0 + r;
    const bool ok = row < n && c * L::kPer < dim && (!PAGED || (unsigned)page < (unsigned)pages);
    const void *pk = zero, *pv = zero;
    if (ok) {
      if constexpr (PAGED) {
        const long long o = ((((long long)page * kv_heads + head) << shift) + (row & ((1 << shift) - 1))) * dim + c * L::kPer;
        pk = k + o; pv = v + o;
      } else {
        pk = k + row * ldk + c * L::kPer; pv = v + row * ldv + c * L::kPer;
      }
    }
    seq_dma16(pk, tk + i * 1024);
    seq_dma16(pv, tv + i * 1024);
  }
};

// One workgroup of W waves: SHARED -- every wave has 32 rows of its own and the waves read the same 64-key tiles; else -- all waves have the
// same 32 rows and each takes 32-key tiles of its own (few rows over many keys), the waves' results are joined through LDS at the end.
template <typename T, int DP, bool PAGED, bool SHARED, int W>
struct Fwd {
  typedef SeqTile<T, DP> L;
  typedef typename SeqVec<T>::v8 v8;
  static constexpr int BN = SHARED ? 64 : 32, NJ = BN / 32;
  static constexpr int BM = SHARED ? 32 * W : 32;
  static constexpr int kTile = BN * L::kRow;                 // bytes of one K or V tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kLds = (SHARED ? 2 : 2 * W) * kStage;
  static constexpr int kIssue = kTile / 1024 / (SHARED ? W : 1);       // transfers of a wave for one tile of K (as many for V)
};

template <typename T, int DP, bool PAGED, bool SHARED, int W>
__global__ void __launch_bounds__(64 * W, (sizeof(T) == 2 && SHARED) ? 2 : 1)
seq_fwd_kernel(const SeqArgs a, const int tiles) {
  typedef Fwd<T, DP, PAGED, SHARED, W> F;
  typedef SeqTile<T, DP> L;
  typedef typename F::v8 v8;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l31 = lane & 31, g = lane >> 5;

  // ---- which rows: packed: one query head, rows = tokens; paged: the heads of a group side by side, rows = (token, head) ------------------------
  const int group = a.heads / a.kv_heads;
  const int mult = PAGED ? group : 1;
  int task = seq_task(blockIdx.x, gridDim.x);
  int kvh, hq, split = 0;
  if (PAGED) { split = task % a.splits; task /= a.splits; hq = 0; kvh = task / tiles; task -= kvh * tiles; }
  else { hq = task % group; task /= group; kvh = task / tiles; task -= kvh * tiles; task = tiles - 1 - task; }     // (causal: the long ones first)
  SeqWhere w;
  if (!seq_find(a.cu_q, a.batch, a.rows_q, mult, F::BM, task, w)) return;
  const int rows = w.n * mult, r0 = w.tile * F::BM;
  int nk, ahead, kstart = 0;                                 // keys of the sequence; keys in front of its first new row
  if (PAGED) {
    const int c = a.ctx[w.b];
    ahead = c < 0 ? 0 : (c > a.max_context ? a.max_context : c);
    const long long room = (long long)a.table_width << a.page_shift;
    nk = ahead + w.n;
    nk = nk > a.max_context ? a.max_context : nk;
    nk = nk > room ? (int)room : nk;
  } else {
    int s = a.cu_k[w.b], e = a.cu_k[w.b + 1];
    s = s < 0 ? 0 : (s > a.rows_k ? a.rows_k : s);
    e = e < s ? s : (e > a.rows_k ? a.rows_k : e);
    kstart = s; nk = e - s; ahead = nk - w.n;
  }
  const int row = r0 + (SHARED ? 32 * wave : 0) + l31;       // this lane's row; both halves of the wave have the same 32
  const bool live = row < rows;
  const int token = w.start + (live ? row / mult : 0), head = kvh * group + (PAGED ? row % mult : hq);
  int limit = 0;                                             // keys this row sees: 0 .. limit - 1
  if (live) { limit = (PAGED || a.causal) ? ahead + row / mult + 1 : nk; limit = limit < 0 ? 0 : (limit > nk ? nk : limit); }
  // the same for the first and the last row of the workgroup (SHARED: and of the wave): tiles behind `some` are not looked at, tiles in
  // front of `all` need no mask
  auto seen = [&](int r) { const int x = (PAGED || a.causal) ? ahead + r / mult + 1 : nk; return x < 0 ? 0 : (x > nk ? nk : x); };
  const int last = (r0 + F::BM < rows ? r0 + F::BM : rows) - 1;
  const int wfirst = SHARED ? r0 + 32 * wave : r0, wlast = (wfirst + 32 < rows ? wfirst + 32 : rows) - 1;
  const int some = seen(last);
  const int wall = wfirst < rows ? seen(wfirst) : nk, wsome = wfirst < rows ? seen(wlast) : 0;
  int k_begin = 0, k_end = some;
  if (PAGED && a.splits > 1) { k_begin = split * a.chunk; k_end = k_begin + a.chunk < some ? k_begin + a.chunk : some; }

  KeySource<T, DP, PAGED> src;
  if (PAGED) { src.k = (const T*)a.k; src.v = (const T*)a.v; src.table = a.table + (size_t)w.b * a.table_width; src.shift = a.page_shift; src.pages = a.pages; }
  else { src.k = (const T*)a.k + kstart * a.ldk + (long long)kvh * a.dim; src.v = (const T*)a.v + kstart * a.ldv + (long long)kvh * a.dim; src.ldk = a.ldk; src.ldv = a.ldv; }
  src.kv_heads = a.kv_heads; src.head = kvh; src.dim = a.dim; src.n = nk; src.zero = a.zero;

  v8 qf[DP / 16];
  {
    const T* qp = (const T*)a.q + token * a.ldq + (long long)head * a.dim;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) qf[t] = seq_load8<T>(qp + 16 * t + 8 * g, live && 16 * t + 8 * g < a.dim);
  }
  f32x16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -__builtin_inff(), l = 0.f;                      // running bound (of the raw products) and this lane's part of the row sum
  const float c = a.scale * kLog2e;

  char* base = smem + (SHARED ? 0 : wave * 2 * F::kStage);
  const int step = SHARED ? F::BN : F::BN * W;
  const int first = k_begin + (SHARED ? 0 : wave * F::BN);
  int pg[F::kIssue];
  auto pages_of = [&](int k0) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < F::kIssue; ++i)
        pg[i] = src.page_of(k0 + ((SHARED ? wave * F::kIssue : 0) + i) * KeySource<T, DP, PAGED>::kRowsOf + lane / L::kChunks);
    }
  };
  auto issue = [&](int k0, int stage) {
    char* t = base + stage * F::kStage;
#pragma unroll
    for (int i = 0; i < F::kIssue; ++i) src.to_lds(k0, (SHARED ? wave * F::kIssue : 0) + i, PAGED ? pg[i] : 0, t, t + F::kTile, lane);
  };
  if (first < k_end) { pages_of(first); issue(first, 0); pages_of(first + step); }
  int stage = 0;
  for (int k0 = first; k0 < k_end; k0 += step, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (SHARED) __syncthreads();                             // this tile is there, and nobody reads the other stage any more
    if (k0 + step < k_end) { issue(k0 + step, stage ^ 1); pages_of(k0 + 2 * step); }
    if (SHARED && k0 >= wsome) continue;
    const char *tk = base + stage * F::kStage, *tv = tk + F::kTile;
    f32x16 s[F::NJ];
#pragma unroll
    for (int j = 0; j < F::NJ; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[j][i] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) s[j] = seq_mma(seq_row<T, DP>(tk, 32 * j + l31, 2 * t + g), qf[t], s[j]);
    }
    if (k0 + F::BN > wall) {                                 // (the wave's first row does not see the whole tile)
#pragma unroll
      for (int j = 0; j < F::NJ; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[j][i] = k0 + 32 * j + 8 * (i >> 2) + 4 * g + (i & 3) < limit ? s[j][i] : -__builtin_inff();
    }
    float mx = s[0][0];
#pragma unroll
    for (int j = 0; j < F::NJ; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[j][i]);
    mx = seq_pair_max(mx);
    if (__builtin_amdgcn_ballot_w64((mx - m) * c > kBound || (mx > m && m == -__builtin_inff()))) {
      const float m1 = fmaxf(m, mx);
      const float f = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m - m1) * c);
      m = m1;
      l *= f;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= f;
    }
    const float mc = m == -__builtin_inff() ? 0.f : m * c;
#pragma unroll
    for (int j = 0; j < F::NJ; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) { s[j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], c, -mc)); l += s[j][i]; }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const v8 p = seq_pack<T>(s[j], t);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[d] = seq_mma(seq_col<T, DP>(tv, 32 * j + 16 * t, d, lane), p, o[d]);
      }
    }
  }
  l = seq_pair_sum(l);

  if (!SHARED) {                                             // the waves' parts of the same rows: wave 0 collects them
    __syncthreads();
    float* x = reinterpret_cast<float*>(smem);               // [W][(DP / 32) * 16 + 2][64]
    constexpr int N = (DP / 32) * 16;
    if (wave > 0) {
      float* y = x + wave * (N + 2) * 64 + lane;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) y[(16 * d + i) * 64] = o[d][i];
      y[N * 64] = m; y[(N + 1) * 64] = l;
    }
    __syncthreads();
    if (wave > 0) return;
    for (int k = 1; k < W; ++k) {
      const float* y = x + k * (N + 2) * 64 + lane;
      const float m2 = y[N * 64], l2 = y[(N + 1) * 64], m1 = fmaxf(m, m2);
      const float f1 = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m - m1) * c), f2 = m2 == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m2 - m1) * c);
      m = m1; l = l * f1 + l2 * f2;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * f1 + y[(16 * d + i) * 64] * f2;
    }
  }
  if (!live) return;
  if (PAGED && a.splits > 1) {
    const long long pr = ((long long)split * a.rows_q + token) * a.heads + head;
    if (g == 0) { a.ml[2 * pr] = m == -__builtin_inff() ? m : m * c; a.ml[2 * pr + 1] = l; }
    float* op = a.part + pr * a.dim;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int col = 32 * d + 8 * (i >> 2) + 4 * g;
        if (col < a.dim && l != 0.f) seq_store4<float>(op + col, o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
      }
    return;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;                // a row that sees nothing: zeros, and minus infinity for its sum
  T* op = (T*)a.out + token * a.ldo + (long long)head * a.dim;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i >> 2) + 4 * g;
      if (col < a.dim) seq_store4<T>(op + col, o[d][i] * inv, o[d][i + 1] * inv, o[d][i + 2] * inv, o[d][i + 3] * inv);
    }
  if (a.lse && g == 0) a.lse[(long long)head * a.rows_q + token] = l != 0.f ? m * a.scale + __logf(l) : -__builtin_inff();
}

// The pieces of a row's keys joined: one wave a row, lanes along the channels.
template <typename T>
__global__ void __launch_bounds__(256) seq_join_kernel(const SeqArgs a) {
  const long long pr = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), n = (long long)a.rows_q * a.heads;
  const int lane = threadIdx.x & 63;
  if (pr >= n) return;
  const int token = (int)(pr / a.heads), head = (int)(pr - (long long)token * a.heads);
  if (token < a.cu_q[0] || token >= a.cu_q[a.batch]) return;         // rows outside the sequences stay as they were
  float m = -__builtin_inff(), l = 0.f;
  if (lane < a.splits) { const sq_f2 x = *reinterpret_cast<const sq_f2*>(a.ml + 2 * (lane * n + pr)); m = x[0]; l = x[1]; }
  if (l == 0.f) m = -__builtin_inff();
  float top = m;
#pragma unroll
  for (int s = 32; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
  const float f = l != 0.f ? __builtin_amdgcn_exp2f(m - top) : 0.f;
  float sum = l * f;
#pragma unroll
  for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s, 64);
  float x0 = 0.f, x1 = 0.f;
  const int col = 2 * lane;
  for (int s = 0; s < a.splits; ++s) {
    const float fs = __shfl(f, s, 64);
    if (fs != 0.f && col < a.dim) {
      const sq_f2 p = *reinterpret_cast<const sq_f2*>(a.part + (s * n + pr) * a.dim + col);
      x0 += fs * p[0]; x1 += fs * p[1];
    }
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  if (col < a.dim) {
    T* op = (T*)a.out + token * a.ldo + (long long)head * a.dim + col;
    op[0] = (T)(x0 * inv); op[1] = (T)(x1 * inv);
  }
  if (a.lse && lane == 0) a.lse[(long long)head * a.rows_q + token] = sum != 0.f ? top * kLn2 + __logf(sum) : -__builtin_inff();
}

int tiles_of(const SeqArgs& a, int mult, int bm) {           // at most: every sequence ends inside a tile
  const long long r = (long long)a.rows_q * mult;
  return (int)(r / bm) + (a.batch < a.rows_q ? a.batch : a.rows_q);
}

template <typename T, int DP, bool PAGED, bool SHARED, int W>
hipError_t fwd(const SeqArgs& a, hipStream_t s) {
  typedef Fwd<T, DP, PAGED, SHARED, W> F;
  static int done[kMaxDevices];
  constexpr int join = SHARED ? 0 : W * ((DP / 32) * 16 + 2) * 256, lds = F::kLds > join ? F::kLds : join;
  opt_in_dynamic_lds((const void*)seq_fwd_kernel<T, DP, PAGED, SHARED, W>, lds, done);
  const int mult = PAGED ? a.heads / a.kv_heads : 1, tiles = tiles_of(a, mult, F::BM);
  const long long grid = (long long)tiles * (PAGED ? (long long)a.kv_heads * a.splits : a.heads);
  if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
  vnr_launch(seq_fwd_kernel<T, DP, PAGED, SHARED, W>, dim3((unsigned)grid), dim3(64 * W), lds, s, a, tiles);
  return hipGetLastError();
}
template <typename T, int DP>
hipError_t fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s) {
  if (!a.table) return fwd<T, DP, false, true, 4>(a, s);
  if (p.shared) return fwd<T, DP, true, true, 4>(a, s);
  return fwd<T, DP, true, false, (sizeof(T) * DP > 256 ? 2 : 4)>(a, s);      // (a wave's four tiles of 32 keys: 64 KiB where a row is 512 bytes)
}
template <typename T> hipError_t fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s) { return a.dim <= 64 ? fwd<T, 64>(a, p, s) : fwd<T, 128>(a, p, s); }
}  // namespace

// Packed prompts have rows enough for the chip.  Over a cache, 32 rows of a sequence or fewer (a decoding step, a short draft): the waves of
// a workgroup take different keys.  The keys are cut where the tiles alone leave compute units idle: about two workgroups for each of them,
// no piece shorter than 256 keys.
SeqPlan seq_plan(const SeqArgs& a, int cus) {
  SeqPlan p;
  if (!a.table) return p;
  const int group = a.heads / a.kv_heads;
  p.shared = (long long)a.max_new * group > 32;
  p.rows = p.shared ? 128 : 32;
  const long long wgs = (long long)tiles_of(a, group, p.rows) * a.kv_heads;
  long long want = wgs > 0 ? (2LL * cus + wgs - 1) / wgs : 1;
  const long long most = (a.max_context + 255) / 256;
  if (want > most) want = most;
  if (want > kMaxSplits) want = kMaxSplits;
  if (want < 1) want = 1;
  const int step = 128;
  p.chunk = (int)(((a.max_context + want - 1) / want + step - 1) / step * step);
  p.splits = p.chunk > 0 ? (a.max_context + p.chunk - 1) / p.chunk : 1;
  if (p.splits < 1) p.splits = 1;
  return p;
}

hipError_t launch_seq_fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s) {
  if (a.dtype == SEQ_F32) return fwd<float>(a, p, s);
  if (a.dtype == SEQ_F16) return fwd<_Float16>(a, p, s);
  return fwd<sq_bf16>(a, p, s);
}
hipError_t launch_seq_join(const SeqArgs& a, hipStream_t s) {
  const long long n = (long long)a.rows_q * a.heads, grid = (n + 3) / 4;
  if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
  if (a.dtype == SEQ_F32) vnr_launch(seq_join_kernel<float>, dim3((unsigned)grid), dim3(256), 0, s, a);
  else if (a.dtype == SEQ_F16) vnr_launch(seq_join_kernel<_Float16>, dim3((unsigned)grid), dim3(256), 0, s, a);
  else vnr_launch(seq_join_kernel<sq_bf16>, dim3((unsigned)grid), dim3(256), 0, s, a);
  return hipGetLastError();
}
}  // namespace vnr
