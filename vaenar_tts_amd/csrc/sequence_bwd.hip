// Attention backward on packed sequences.  With P = exp(scale S - lse), dP = dO V', delta_i = sum_d dO_id O_id:
//   dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS' Q,  dV = P' dO.
// Two kernels, each the owner of what it writes (no atomics: the same bits every time, and the heads of a group are summed inside the
// workgroup that owns their keys): seq_dq_kernel goes over the keys of its 128 query rows, seq_dkv_kernel over the query rows (of every head
// of the group) of its 128 keys.  Both rebuild S and dP -- seven products instead of the five that one pass with atomics onto dQ would take.
// P and dS are rounded to the operands' type for the products that read them; every sum is held in 32 bits.
#include "sequence.h"

namespace vnr {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

template <typename T, int DP>
__device__ __forceinline__ void tile_to_lds(const T* base, long long ld, int r0, int n, int dim, int i, char* tile, int lane, const void* zero) {
  typedef SeqTile<T, DP> L;
  constexpr int kRowsOf = 64 / L::kChunks;
  const int r = i * kRowsOf + lane / L::kChunks, c = (lane % L::kChunks) ^ (r & 7), row = r0 + r;
  const void* p = (row < n && c * L::kPer < dim) ? (const void*)(base + row * ld + c * L::kPer) : zero;
  seq_dma16(p, tile + i * 1024);
}
__device__ __forceinline__ void clamped(const int32_t* cu, int b, int total, int& start, int& n) {
  int s = cu[b], e = cu[b + 1];
  s = s < 0 ? 0 : (s > total ? total : s);
  e = e < s ? s : (e > total ? total : e);
  start = s; n = e - s;
}

// 128 query rows of one head.  Leaves delta and lse log2 e of its rows for the other kernel: delta [2][heads][rows_q].
template <typename T, int DP>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) seq_dq_kernel(const SeqGradArgs ga, const int tiles) {
  typedef SeqTile<T, DP> L;
  typedef typename SeqVec<T>::v8 v8;
  const SeqArgs& a = ga.f;
  constexpr int BN = 64, kTile = BN * L::kRow, kStage = 2 * kTile, kIssue = kTile / 4096;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l31 = lane & 31, g = lane >> 5;
  const int group = a.heads / a.kv_heads;
  int task = seq_task(blockIdx.x, gridDim.x);
  const int hq = task % group; task /= group;
  const int kvh = task / tiles; task = tiles - 1 - (task - kvh * tiles);
  SeqWhere w;
  if (!seq_find(a.cu_q, a.batch, a.rows_q, 1, 128, task, w)) return;
  int ks, nk;
  clamped(a.cu_k, w.b, a.rows_k, ks, nk);
  const int ahead = nk - w.n, head = kvh * group + hq;
  const int r0 = w.tile * 128, row = r0 + 32 * wave + l31;
  const bool live = row < w.n;
  const int token = w.start + (live ? row : 0);
  auto seen = [&](int r) { const int x = a.causal ? ahead + r + 1 : nk; return x < 0 ? 0 : (x > nk ? nk : x); };
  const int limit = live ? seen(row) : 0;
  const int last = (r0 + 128 < w.n ? r0 + 128 : w.n) - 1, some = seen(last);
  const int wfirst = r0 + 32 * wave, wlast = (wfirst + 32 < w.n ? wfirst + 32 : w.n) - 1;
  const int wall = wfirst < w.n ? seen(wfirst) : nk, wsome = wfirst < w.n ? seen(wlast) : 0;

  v8 qf[DP / 16], df[DP / 16];
  float delta = 0.f;
  {
    const long long ho = (long long)head * a.dim;
    const T *qp = (const T*)a.q + token * a.ldq + ho, *dp = (const T*)ga.dout + token * ga.lddo + ho, *op = (const T*)a.out + token * a.ldo + ho;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      const int e0 = 16 * t + 8 * g;
      const bool ok = live && e0 < a.dim;
      qf[t] = seq_load8<T>(qp + e0, ok);
      df[t] = seq_load8<T>(dp + e0, ok);
      const v8 o = seq_load8<T>(op + e0, ok);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)df[t][e] * (float)o[e];
    }
    delta = seq_pair_sum(delta);
  }
  float lse2 = 0.f;
  if (live) {
    const long long at = (long long)head * a.rows_q + token, plane = (long long)a.heads * a.rows_q;
    lse2 = a.lse[at] * kLog2e;
    if (g == 0) { ga.delta[at] = delta; ga.delta[plane + at] = lse2; }
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  const float c = a.scale * kLog2e;
  const T *kb = (const T*)a.k + ks * a.ldk + (long long)kvh * a.dim, *vb = (const T*)a.v + ks * a.ldv + (long long)kvh * a.dim;
  auto issue = [&](int k0, int stage) {
    char* t = smem + stage * kStage;
#pragma unroll
    for (int i = 0; i < kIssue; ++i) {
      tile_to_lds<T, DP>(kb, a.ldk, k0, nk, a.dim, wave * kIssue + i, t, lane, a.zero);
      tile_to_lds<T, DP>(vb, a.ldv, k0, nk, a.dim, wave * kIssue + i, t + kTile, lane, a.zero);
    }
  };
  if (some > 0) issue(0, 0);
  int stage = 0;
  for (int k0 = 0; k0 < some; k0 += BN, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (k0 + BN < some) issue(k0 + BN, stage ^ 1);
    if (k0 >= wsome) continue;
    const char *tk = smem + stage * kStage, *tv = tk + kTile;
    const bool masked = k0 + BN > wall;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x16 s, p;
#pragma unroll
      for (int i = 0; i < 16; ++i) { s[i] = 0.f; p[i] = 0.f; }
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) {
        s = seq_mma(seq_row<T, DP>(tk, 32 * j + l31, 2 * t + g), qf[t], s);
        p = seq_mma(seq_row<T, DP>(tv, 32 * j + l31, 2 * t + g), df[t], p);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -lse2)) * (p[i] - delta);
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = k0 + 32 * j + 8 * (i >> 2) + 4 * g + (i & 3) < limit ? s[i] : 0.f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const v8 ds = seq_pack<T>(s, t);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) acc[d] = seq_mma(seq_col<T, DP>(tk, 32 * j + 16 * t, d, lane), ds, acc[d]);
      }
    }
  }
  if (!live) return;
  T* dq = (T*)ga.dq + token * ga.lddq + (long long)head * a.dim;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i >> 2) + 4 * g;
      if (col < a.dim) seq_store4<T>(dq + col, acc[d][i] * a.scale, acc[d][i + 1] * a.scale, acc[d][i + 2] * a.scale, acc[d][i + 3] * a.scale);
    }
}

// 128 keys of one key / value head: 32 a wave, as the columns of S = Q K' and dP = dO V'; the query rows of every head of the group pass
// through LDS in tiles of BQ.
template <typename T, int DP, int BQ>
__global__ void __launch_bounds__(256, 1) seq_dkv_kernel(const SeqGradArgs ga, const int tiles) {
  typedef SeqTile<T, DP> L;
  typedef typename SeqVec<T>::v8 v8;
  const SeqArgs& a = ga.f;
  constexpr int kTile = BQ * L::kRow, kStage = 2 * kTile + 2 * BQ * 4, kIssue = kTile / 4096;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l31 = lane & 31, g = lane >> 5;
  const int group = a.heads / a.kv_heads;
  int task = seq_task(blockIdx.x, gridDim.x);
  const int kvh = task / tiles; task -= kvh * tiles;         // (causal: the first keys of a sequence are seen by most rows: long ones first)
  SeqWhere w;
  if (!seq_find(a.cu_k, a.batch, a.rows_k, 1, 128, task, w)) return;
  int qs, nq;
  clamped(a.cu_q, w.b, a.rows_q, qs, nq);
  const int nk = w.n, ahead = nk - nq;
  const int k0 = w.tile * 128, kw = k0 + 32 * wave, key = kw + l31;
  const bool live = key < nk;
  v8 kf[DP / 16], vf[DP / 16];
  {
    const int at = w.start + (live ? key : 0);
    const T *kp = (const T*)a.k + at * a.ldk + (long long)kvh * a.dim, *vp = (const T*)a.v + at * a.ldv + (long long)kvh * a.dim;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      const int e0 = 16 * t + 8 * g;
      kf[t] = seq_load8<T>(kp + e0, live && e0 < a.dim);
      vf[t] = seq_load8<T>(vp + e0, live && e0 < a.dim);
    }
  }
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) { dk[d][i] = 0.f; dv[d][i] = 0.f; }
  const float c = a.scale * kLog2e;
  // rows in front of `first` see none of the workgroup's keys
  int first = a.causal ? k0 - ahead : 0;
  first = first < 0 ? 0 : first / BQ * BQ;
  const int per = nq > first ? (nq - first + BQ - 1) / BQ : 0, total = per * group;
  const long long plane = (long long)a.heads * a.rows_q;
  auto issue = [&](int it, int stage) {
    const int h = kvh * group + it / per, q0 = first + it % per * BQ;
    char* t = smem + stage * kStage;
    const T *qb = (const T*)a.q + qs * a.ldq + (long long)h * a.dim, *db = (const T*)ga.dout + qs * ga.lddo + (long long)h * a.dim;
#pragma unroll
    for (int i = 0; i < kIssue; ++i) {
      tile_to_lds<T, DP>(qb, a.ldq, q0, nq, a.dim, wave * kIssue + i, t, lane, a.zero);
      tile_to_lds<T, DP>(db, ga.lddo, q0, nq, a.dim, wave * kIssue + i, t + kTile, lane, a.zero);
    }
    if (wave < 2 && lane < BQ) {                             // delta and lse of the rows: four bytes a lane
      const float* x = ga.delta + wave * plane + (long long)h * a.rows_q + qs + q0 + lane;
      const void* p = q0 + lane < nq ? (const void*)x : a.zero;
      __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)(t + 2 * kTile + wave * BQ * 4), 4, 0, 0);
    }
  };
  if (total > 0) issue(0, 0);
  int stage = 0;
  for (int it = 0; it < total; ++it, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (it + 1 < total) issue(it + 1, stage ^ 1);
    const int q0 = first + it % per * BQ;
    const char *tq = smem + stage * kStage, *td = tq + kTile;
    const float *delta = reinterpret_cast<const float*>(td + kTile), *lse2 = delta + BQ;
#pragma unroll
    for (int j = 0; j < BQ / 32; ++j) {
      const int r0 = q0 + 32 * j;
      if (a.causal && r0 + 31 + ahead < kw) continue;        // (wave-uniform) none of these rows sees the wave's keys
      f32x16 s, p;
#pragma unroll
      for (int i = 0; i < 16; ++i) { s[i] = 0.f; p[i] = 0.f; }
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) {
        s = seq_mma(seq_row<T, DP>(tq, 32 * j + l31, 2 * t + g), kf[t], s);
        p = seq_mma(seq_row<T, DP>(td, 32 * j + l31, 2 * t + g), vf[t], p);
      }
      const bool masked = a.causal && r0 + ahead < kw + 31;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const sq_f4 ls = *reinterpret_cast<const sq_f4*>(lse2 + 32 * j + 8 * q + 4 * g), de = *reinterpret_cast<const sq_f4*>(delta + 32 * j + 8 * q + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * q + e;
          float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -ls[e])), y = x * (p[i] - de[e]);
          if (masked) { const bool ok = key <= r0 + 8 * q + 4 * g + e + ahead; x = ok ? x : 0.f; y = ok ? y : 0.f; }
          s[i] = x; p[i] = y;
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const v8 pf = seq_pack<T>(s, t), sf = seq_pack<T>(p, t);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          dv[d] = seq_mma(seq_col<T, DP>(td, 32 * j + 16 * t, d, lane), pf, dv[d]);
          dk[d] = seq_mma(seq_col<T, DP>(tq, 32 * j + 16 * t, d, lane), sf, dk[d]);
        }
      }
    }
  }
  if (!live) return;
  T *pk = (T*)ga.dk + (w.start + key) * ga.lddk + (long long)kvh * a.dim, *pv = (T*)ga.dv + (w.start + key) * ga.lddv + (long long)kvh * a.dim;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i >> 2) + 4 * g;
      if (col < a.dim) {
        seq_store4<T>(pk + col, dk[d][i] * a.scale, dk[d][i + 1] * a.scale, dk[d][i + 2] * a.scale, dk[d][i + 3] * a.scale);
        seq_store4<T>(pv + col, dv[d][i], dv[d][i + 1], dv[d][i + 2], dv[d][i + 3]);
      }
    }
}

template <typename T, int DP> hipError_t grad(const SeqGradArgs& a, hipStream_t s) {
  typedef SeqTile<T, DP> L;
  static int done_q[kMaxDevices], done_kv[kMaxDevices];
  const SeqArgs& f = a.f;
  if (f.rows_q > 0) {
    constexpr int lds = 2 * 2 * 64 * L::kRow;
    opt_in_dynamic_lds((const void*)seq_dq_kernel<T, DP>, lds, done_q);
    const int tiles = f.rows_q / 128 + (f.batch < f.rows_q ? f.batch : f.rows_q);
    const long long grid = (long long)tiles * f.heads;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    vnr_launch(seq_dq_kernel<T, DP>, dim3((unsigned)grid), dim3(256), lds, s, a, tiles);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (f.rows_k > 0) {
    constexpr int BQ = 64, lds = 2 * (2 * BQ * L::kRow + 8 * BQ);
    static_assert(lds <= 160 * 1024, "LDS");
    opt_in_dynamic_lds((const void*)seq_dkv_kernel<T, DP, BQ>, lds, done_kv);
    const int tiles = f.rows_k / 128 + (f.batch < f.rows_k ? f.batch : f.rows_k);
    const long long grid = (long long)tiles * f.kv_heads;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    vnr_launch(seq_dkv_kernel<T, DP, BQ>, dim3((unsigned)grid), dim3(256), lds, s, a, tiles);
  }
  return hipGetLastError();
}
template <typename T> hipError_t grad(const SeqGradArgs& a, hipStream_t s) { return a.f.dim <= 64 ? grad<T, 64>(a, s) : grad<T, 128>(a, s); }
}  // namespace

hipError_t launch_seq_grad(const SeqGradArgs& a, hipStream_t s) {
  if (a.f.dtype == SEQ_F32) return grad<float>(a, s);
  if (a.f.dtype == SEQ_F16) return grad<_Float16>(a, s);
  return grad<sq_bf16>(a, s);
}
}  // namespace vnr
