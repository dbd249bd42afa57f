// Attention backward on packed sequences.  With P = exp(scale S - lse), dP = dO V', delta_i = sum_d dO_id O_id:
//   dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS' Q,  dV = P' dO.
// Two kernels, each the owner of what it writes (no atomics: the same bits every time, and the heads of a group are summed inside the
// workgroup that owns their keys): seq_dq_kernel goes over the keys of its query rows, seq_dkv_kernel over the query rows (of every head
// of the group) of its keys.  Both rebuild S and dP -- seven products instead of the five that one pass with atomics onto dQ would take.
// P is rounded once to the operands' type for dV (as dout is); what that rounding leaves of dS goes through a second product in 16-bit types --
// the differences dP - delta cancel, and a rounding of what is left shows in dQ and dK (with it they are within 1.01 of the error of a plain
// form in 32 bits whose results are rounded once, dV within 1.4).  Every sum is held in 32 bits.
// float16 holds 2^-24 .. 65504, dS anything (dout of 1e-4 over 2000 keys is below, dout of 1500 above): it is multiplied by a power of two
// that fits the largest of its row (dQ) or key (dK) so far, a running bound as the forward's of the logits, and the sums are divided by it at the end.
// P needs no such search, it is at most 1 (and held there: under large logits the rounding of lse puts it above): 2^15 P goes into dV's product
// (weights below 2^-40 are lost, those from 2^-29 on are rounded like any other).
//
// What bounds it: 4 sequences of up to 2048 rows, 32 heads over 8 of 128, bf16, causal: 254 - 265 us by card -- nine products where the formulas have
// five, 0.79 PFLOP/s of them; a workgroup of dK and dV lasts as long as the rows that see its keys (the matrix pipe is busy 29 % of its cycles, 40 % of
// dQ's).  32 utterances of up to 400 rows, 4 heads of 64, f32: 113 us, the 32-bit matrix instructions' rate (the pipe is busy 22 and 24 %: about one
// wave a SIMD) and LDS reads of four bytes a lane.  (Under a profiler, which runs every kernel alone and at other clocks: 107 us for dQ and 171 for
// dK and dV, 52 and 66.)
#include "sequence.h"

namespace vnr {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
template <typename T> struct Weight { static constexpr float kLift = __is_same(T, _Float16) ? 15.f : 0.f, kTimes = __is_same(T, _Float16) ? 32768.f : 1.f; };      // of P in dV's product

// Rows of one head in memory, `ld` bytes apart; rows from n on read as zeros.  Whole tiles go by scalar addresses, the last one of a sequence
// and heads narrower than the tile by an address in every lane (zeros where there is nothing).
template <typename T, int DP> struct Rows {                    // (`first` is the same in set and fetch)
  typedef SeqTile<T, DP> L;
  typedef SeqLanes<T, DP> W;
  long long ld; int n, dim; const void* zero; bool plain; W w;
  __device__ __forceinline__ void set(long long stride, int rows, int width, const void* zeros, int lane, int first) {
    ld = stride * (int)sizeof(T); n = rows; dim = width; zero = zeros;
    plain = width == DP && stride < (1 << 24) && !(ld % L::kRow);      // (SeqLanes; a lane's offset in 32 bits)
    w.set((unsigned)ld, lane, first);
  }
  // transfers first .. first + N - 1 of the tile of `rows` rows that starts at row r0 of `base`
  template <int N> __device__ __forceinline__ void fetch(const void* base, int r0, int rows, int first, unsigned dst, int lane) const {
    const char* p = (const char*)base + (r0 + first * W::kRowsOf) * ld;
    if (plain && r0 + rows <= n) {
#pragma unroll
      for (int i = 0; i < N; ++i) seq_dma16(p + i * W::kRowsOf * ld, w.at(i), dst + (first + i) * 1024);
      return;
    }
    asm volatile("" : "+v"(lane));                           // (opaque: or what follows from it is kept in registers all the way)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = lane / L::kChunks, c = (lane % L::kChunks) ^ L::turn((first + i) * W::kRowsOf + r);
      const char* q = p + (i * W::kRowsOf + r) * ld + c * 16;
      seq_dma16(r0 + (first + i) * W::kRowsOf + r < n && c * L::kPer < dim ? (const void*)q : zero, dst + (first + i) * 1024);
    }
  }
};

// The columns of dS as float16 operands: x holds 2^lift of them, and where that passes 2^15 the column's lift comes down to where its largest is
// 2^10 .. 2^11 -- `acc`, what went through the second product before, with it.  (What the second half's smallest step, 2^-25, leaves out is 2^-35 of a
// column's largest.  Both lanes of a column, 32 apart, take the same turn; a value that is not finite moves nothing.  In float16 the bf16 case above
// takes 275 us with it, 261 without, the f32 one 41 and 38.)
constexpr int kFirst = 60;                                   // at first: 2^60 times 2^15 P times what float16 operands make of dP stays a 32-bit number
template <int N> __device__ __forceinline__ void fit(f32x16& x, int& lift, f32x16 (&acc)[N]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, __builtin_fabsf(x[i]));
  top = seq_pair_max(top);
  if (__builtin_amdgcn_ballot_w64(top > 32768.f)) {
    const int e = 11 - __builtin_amdgcn_frexp_expf(top), down = top > 32768.f && e < 0 ? e : 0;
    lift += down;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_ldexpf(x[i], down);
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = __builtin_amdgcn_ldexpf(acc[d][i], down);
  }
}

// 32 RG query rows of one head; KS key groups of waves, as in the forward kernel.  Leaves delta and lse log2 e of its rows (less the lift of their
// weights) for the other kernel: delta [2][heads][rows_q].
template <typename T, int DP, int RG, int KS>
__global__ void __launch_bounds__(64 * RG * KS, sizeof(T) == 2 ? 2 : 1) seq_dq_kernel(const SeqGradArgs ga, const int tiles) {
  typedef SeqTile<T, DP> L;
  typedef typename SeqVec<T>::v8 v8;
  const SeqArgs& a = ga.f;
  constexpr int BM = 32 * RG, BN = RG == 4 ? 64 : 32, kTile = BN * L::kRow, kStage = 2 * kTile, kIssue = kTile / 1024 / RG, step = BN * KS;
  extern __shared__ __attribute__((aligned(512))) char smem[];         // (SeqReads: tiles start at multiples of their row)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % RG, kg = wave / RG, l31 = lane & 31, g = lane >> 5;
  const int group = a.heads / a.kv_heads;
  int task = seq_task(blockIdx.x, gridDim.x);
  const int hq = task % group; task /= group;
  const int kvh = task / tiles; task -= kvh * tiles;
  SeqWhere w;
  if (!seq_find(a.cu_q, a.batch, a.rows_q, 1, BM, task, a.cu_k, 1, w)) return;
  int ks, nk;
  seq_clamp(w.x0, w.x1, a.rows_k, ks, nk);
  const int ahead = nk - w.n, head = kvh * group + hq;
  const int r0 = ((w.n + BM - 1) / BM - 1 - w.tile) * BM, row = r0 + 32 * rg + l31;
  const bool live = row < w.n;
  const int token = w.start + (live ? row : 0);
  auto seen = [&](int r) { const int x = a.causal ? ahead + r + 1 : nk; return x < 0 ? 0 : (x > nk ? nk : x); };
  const int limit = live ? seen(row) : 0;
  const int last = (r0 + BM < w.n ? r0 + BM : w.n) - 1, some = seen(last);
  const int wfirst = r0 + 32 * rg, wlast = (wfirst + 32 < w.n ? wfirst + 32 : w.n) - 1;
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
      qf[t] = seq_load8<T>(qp + e0, ok, a.zero);
      df[t] = seq_load8<T>(dp + e0, ok, a.zero);
      const v8 o = seq_load8<T>(op + e0, ok, a.zero);
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)df[t][e] * (float)o[e];
    }
    delta = seq_pair_sum(delta);
  }
  float lse2 = 0.f;
  const long long place = (long long)head * a.rows_q + token;
  if (live) lse2 = a.lse[place] * kLog2e;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
  const float c = a.scale * kLog2e;
  const T *kb = (const T*)a.k + ks * a.ldk + (long long)kvh * a.dim, *vb = (const T*)a.v + ks * a.ldv + (long long)kvh * a.dim;
  const unsigned lds = seq_lds(smem) + kg * 2 * kStage;
  SeqReads<T, DP> reads;
  reads.set(lane);
  Rows<T, DP> rk, rv;
  rk.set(a.ldk, nk, a.dim, a.zero, lane, rg * kIssue); rv.set(a.ldv, nk, a.dim, a.zero, lane, rg * kIssue);
  seq_settle(qf); seq_settle(df);
  auto products = [&](unsigned tk, int j, f32x16& s, f32x16& p) {
#pragma unroll
    for (int i = 0; i < 16; ++i) { s[i] = 0.f; p[i] = 0.f; }
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      s = seq_mma(seq_row<T, DP>(tk, 32 * j, t), qf[t], s);
      p = seq_mma(seq_row<T, DP>(tk, BN + 32 * j, t), df[t], p);           // (V lies behind K)
    }
  };
  // The rounding of `out` reaches dS through delta, and where few keys share a row's weight nothing averages it away (rows of two keys: dQ twice as
  // far from 64 bits as a plain form's, of eight 1.2 times).  Rows that see up to 64 keys take delta = sum_j P dP instead, in turns of their own
  // over these keys: whole short sequences, of a causal one the workgroup that holds its first rows.
  constexpr int kFew = 64;
  if (sizeof(T) == 2 && seen(r0) <= kFew) {
    float sum = 0.f;
    const int end = some < kFew ? some : kFew;
    for (int kt = -BN, stage = 0; kt < end; kt += BN, stage ^= kStage) {
      seq_dma_wait();
      __syncthreads();
      if (kt + BN < end) {
        const unsigned t = lds + (stage ^ kStage);
        rk.template fetch<kIssue>(kb, kt + BN, BN, rg * kIssue, t, lane);
        rv.template fetch<kIssue>(vb, kt + BN, BN, rg * kIssue, t + kTile, lane);
      }
      if (kt < 0 || kt >= wsome) continue;
      const unsigned tk = seq_at(lds + stage, reads.row);
#pragma unroll
      for (int j = 0; j < BN / 32; ++j) {
        f32x16 s, p;
        products(tk, j, s, p);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -lse2)) * p[i];
          sum += kt + 32 * j + 8 * (i >> 2) + 4 * g + (i & 3) < limit ? x : 0.f;
        }
      }
    }
    sum = seq_pair_sum(sum);
    delta = limit <= kFew ? sum : delta;
  }
  if (live && g == 0 && kg == 0) { ga.delta[place] = delta; ga.delta[(long long)a.heads * a.rows_q + place] = lse2 - Weight<T>::kLift; }
  constexpr bool kFit = __is_same(T, _Float16);
  int lift = kFit ? kFirst : 0;
  int k0 = (kg - KS) * BN, stage = 0;                        // (the first turn only fetches)
  for (int kt = -step; kt < some; kt += step, k0 += step, stage ^= kStage) {
    seq_dma_wait();
    __syncthreads();
    if (k0 + step < some) {
      const unsigned t = lds + (stage ^ kStage);
      rk.template fetch<kIssue>(kb, k0 + step, BN, rg * kIssue, t, lane);
      rv.template fetch<kIssue>(vb, k0 + step, BN, rg * kIssue, t + kTile, lane);
    }
    if (kt < 0 || k0 >= some || k0 >= wsome) continue;
    const unsigned tk = seq_at(lds + stage, reads.row), tc = seq_at(lds + stage, reads.col);
    const bool masked = k0 + BN > wall;
#pragma unroll
    for (int j = 0; j < BN / 32; ++j) {
      f32x16 s, p;
      products(tk, j, s, p);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -lse2));
        s[i] = x * (kFit ? __builtin_amdgcn_ldexpf(p[i] - delta, lift) : p[i] - delta);
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = k0 + 32 * j + 8 * (i >> 2) + 4 * g + (i & 3) < limit ? s[i] : 0.f;
      }
      if constexpr (kFit) fit(s, lift, acc);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (sizeof(T) == 2) {
          v8 rest;
          const v8 ds = seq_pack<T>(s, t, rest);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) {
            const v8 k = seq_col<T, DP>(tc, 32 * j + 16 * t, d);
            acc[d] = seq_mma(k, ds, acc[d]);
            acc[d] = seq_mma(k, rest, acc[d]);
          }
        } else {
          const v8 ds = seq_pack<T>(s, t);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) acc[d] = seq_mma(seq_col<T, DP>(tc, 32 * j + 16 * t, d), ds, acc[d]);
        }
      }
    }
  }
  if constexpr (kFit) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = __builtin_amdgcn_ldexpf(acc[d][i], -lift);
  }
  if (KS > 1) {                                              // the key groups' parts of the same rows, summed in the groups' order
    __syncthreads();
    constexpr int N = (DP / 32) * 16;
    float* x = reinterpret_cast<float*>(smem) + lane;
    if (kg > 0) {
      float* y = x + ((kg - 1) * RG + rg) * N * 64;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) y[(16 * d + i) * 64] = acc[d][i];
    }
    __syncthreads();
    if (kg > 0) return;
    for (int k = 0; k < KS - 1; ++k) {
      const float* y = x + (k * RG + rg) * N * 64;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] += y[(16 * d + i) * 64];
    }
  }
  if (!live) return;
  const float out = limit == 1 ? 0.f : a.scale;              // one key: its weight is 1 whatever the logit, dQ is exactly nothing (not a rounding of delta)
  T* dq = (T*)ga.dq + token * ga.lddq + (long long)head * a.dim;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i >> 2) + 4 * g;
      if (col < a.dim) seq_store4<T>(dq + col, acc[d][i] * out, acc[d][i + 1] * out, acc[d][i + 2] * out, acc[d][i + 3] * out);
    }
}

// 32 KG keys of one key / value head, 32 a wave, as the columns of S = Q K' and dP = dO V'; the query rows of every head of the group pass
// through LDS in tiles of 32.  HG row groups of waves take the tiles in turn (each with buffers of its own) and their sums are joined at the
// end: a sequence's first keys are seen by all of its rows in every head, one wave for them would outlast the rest of the launch.
template <typename T, int DP, int KG, int HG>
__global__ void __launch_bounds__(64 * KG * HG, HG == 4 || sizeof(T) * DP == 128 ? 2 : 1) seq_dkv_kernel(const SeqGradArgs ga, const int tiles) {
  typedef SeqTile<T, DP> L;
  typedef typename SeqVec<T>::v8 v8;
  const SeqArgs& a = ga.f;
  constexpr int BK = 32 * KG, BQ = 32, kTile = BQ * L::kRow, kStage = 2 * kTile + (L::kRow > 256 ? 512 : 256), kIssue = kTile / 1024 / KG;
  extern __shared__ __attribute__((aligned(512))) char smem[];         // (SeqReads: tiles start at multiples of their row)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave % KG, hg = wave / KG, l31 = lane & 31, g = lane >> 5;
  const int group = a.heads / a.kv_heads;
  int task = seq_task(blockIdx.x, gridDim.x);
  const int kvh = task / tiles; task -= kvh * tiles;         // (causal: the first keys of a sequence are seen by most rows: long ones first)
  SeqWhere w;
  if (!seq_find(a.cu_k, a.batch, a.rows_k, 1, BK, task, a.cu_q, 1, w)) return;
  int qs, nq;
  seq_clamp(w.x0, w.x1, a.rows_q, qs, nq);
  const int nk = w.n, ahead = nk - nq;
  // The first keys of a sequence are seen by most rows.  Two workgroups share a compute unit, the second of them about a sequence further in
  // the tasks' order: every other sequence goes from its light end, so that a heavy one meets a light one.
  const int k0 = (w.rank & 1 ? (nk + BK - 1) / BK - 1 - w.tile : w.tile) * BK, kw = k0 + 32 * kg, key = kw + l31;
  const bool live = key < nk;
  v8 kf[DP / 16], vf[DP / 16];
  {
    const int at = w.start + (live ? key : 0);
    const T *kp = (const T*)a.k + at * a.ldk + (long long)kvh * a.dim, *vp = (const T*)a.v + at * a.ldv + (long long)kvh * a.dim;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      const int e0 = 16 * t + 8 * g;
      kf[t] = seq_load8<T>(kp + e0, live && e0 < a.dim, a.zero);
      vf[t] = seq_load8<T>(vp + e0, live && e0 < a.dim, a.zero);
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
  const unsigned lds = seq_lds(smem) + hg * 2 * kStage;
  Rows<T, DP> rq, rd;
  rq.set(a.ldq, nq, a.dim, a.zero, lane, kg * kIssue); rd.set(ga.lddo, nq, a.dim, a.zero, lane, kg * kIssue);
  const char *qb = (const char*)((const T*)a.q + qs * a.ldq), *db = (const char*)((const T*)ga.dout + qs * ga.lddo);
  seq_settle(kf); seq_settle(vf);
  // ---- one tile of rows: the two products, the weights and their gradients, what they add to dV and dK ----------------------------------------
  f32x16 s, p;
  constexpr bool kFit = __is_same(T, _Float16);
  int lift = kFit ? kFirst : 0;
  SeqReads<T, DP> reads;
  reads.set(lane);
  auto products = [&](unsigned tile) {
    const unsigned at = seq_at(tile, reads.row);
#pragma unroll
    for (int i = 0; i < 16; ++i) { s[i] = 0.f; p[i] = 0.f; }
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
      s = seq_mma(seq_row<T, DP>(at, 0, t), kf[t], s);
      p = seq_mma(seq_row<T, DP>(at, BQ, t), vf[t], p);      // (dO lies behind Q)
    }
  };
  auto weights = [&](unsigned tile) {
    const unsigned at = seq_at(tile, 16 * g);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const sq_f4 de = seq_ds<sq_f4>(at + 2 * kTile + 32 * q), ls = seq_ds<sq_f4>(at + 2 * kTile + 4 * BQ + 32 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * q + e;
        float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -ls[e]));
        if constexpr (kFit) x = __builtin_elementwise_minimum(x, Weight<T>::kTimes);         // (NaN stays NaN)
        p[i] = x * (kFit ? __builtin_amdgcn_ldexpf(p[i] - de[e], lift) : p[i] - de[e]);
        s[i] = x;
      }
    }
  };
  auto masks = [&](int row) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int sees = row + 8 * (i >> 2) + 4 * g + (i & 3) + ahead;
      const float f = sees == 0 ? 0.f : p[i];                // (the row that sees key 0 alone adds exactly nothing to dK)
      s[i] = key <= sees ? s[i] : 0.f; p[i] = key <= sees ? f : 0.f;
    }
  };
  auto sums = [&](unsigned tile) {
    const unsigned at = seq_at(tile, reads.col);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      v8 rest = {};
      const v8 pf = seq_pack<T>(s, t);
      v8 sf;
      if constexpr (sizeof(T) == 2) sf = seq_pack<T>(p, t, rest); else sf = seq_pack<T>(p, t);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        dv[d] = seq_mma(seq_col<T, DP>(at, BQ + 16 * t, d), pf, dv[d]);
        const v8 q = seq_col<T, DP>(at, 16 * t, d);
        dk[d] = seq_mma(q, sf, dk[d]);
        if constexpr (sizeof(T) == 2) dk[d] = seq_mma(q, rest, dk[d]);
      }
    }
  };
  // tile `at` of head `h` of the group is fetched next
  int h = 0, at = hg;
  while (per > 0 && at >= per) { at -= per; ++h; }
  auto fetch = [&](int stage) {
    const unsigned t = lds + stage;
    const int hd = kvh * group + h, r0 = first + at * BQ;
    const long long ho = (long long)hd * a.dim * (int)sizeof(T);
    rq.template fetch<kIssue>(qb + ho, r0, BQ, kg * kIssue, t, lane);
    rd.template fetch<kIssue>(db + ho, r0, BQ, kg * kIssue, t + kTile, lane);
    if (kg == 0) {                                           // delta, then lse of the tile's rows: four bytes a lane
      const float* x = ga.delta + (g ? plane : 0) + (long long)hd * a.rows_q + qs + r0 + l31;
      seq_dma4(r0 + l31 < nq ? (const void*)x : a.zero, t + 2 * kTile);
    }
    at += HG;
    while (at >= per) { at -= per; ++h; }
    return r0;
  };
  auto sees = [&](int row) { return !a.causal || row + 31 + ahead >= kw; };    // does any row of the tile see the wave's keys?
  int r0 = 0, stage = 0;                                   // the first turn only fetches
  for (int turn = -HG; turn < total; turn += HG, stage ^= kStage) {          // (every group as often: the barrier is everybody's)
    const int it = turn + hg, row = r0;
    seq_dma_wait();
    if (KG > 1) __syncthreads();
    if (it + HG < total) r0 = fetch(stage ^ kStage);
    if (turn < 0 || it >= total || !sees(row)) continue;
    products(lds + stage);
    weights(lds + stage);
    if (a.causal && row + ahead < kw + 31) masks(row);
    if constexpr (kFit) fit(p, lift, dk);
    sums(lds + stage);
  }
  if constexpr (kFit) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) { dk[d][i] = __builtin_amdgcn_ldexpf(dk[d][i], -lift - (int)Weight<T>::kLift); dv[d][i] *= 1.f / Weight<T>::kTimes; }
  }
  if (HG > 1) {                                              // the row groups' sums, in their order: dK, then dV through the same buffer
    constexpr int N = (DP / 32) * 16;
    float* x = reinterpret_cast<float*>(smem) + lane;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
      if (hg > 0) {
        float* y = x + ((hg - 1) * KG + kg) * N * 64;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) y[(16 * d + i) * 64] = half ? dv[d][i] : dk[d][i];
      }
      __syncthreads();
      if (hg == 0) {
        for (int k = 0; k < HG - 1; ++k) {
          const float* y = x + (k * KG + kg) * N * 64;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) { if (half) dv[d][i] += y[(16 * d + i) * 64]; else dk[d][i] += y[(16 * d + i) * 64]; }
        }
      }
    }
    if (hg > 0) return;
  }
  if (!live) return;
  const float out = nk == 1 ? 0.f : a.scale;                 // (as in dQ)
  T *pk = (T*)ga.dk + (w.start + key) * ga.lddk + (long long)kvh * a.dim, *pv = (T*)ga.dv + (w.start + key) * ga.lddv + (long long)kvh * a.dim;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i >> 2) + 4 * g;
      if (col < a.dim) {
        seq_store4<T>(pk + col, dk[d][i] * out, dk[d][i + 1] * out, dk[d][i + 2] * out, dk[d][i + 3] * out);
        seq_store4<T>(pv + col, dv[d][i], dv[d][i + 1], dv[d][i + 2], dv[d][i + 3]);
      }
    }
}

// tiles of `rows` rows, at most: every sequence ends inside one
long long tiles_of(int total, int batch, int rows) { return total / rows + (batch < total ? batch : total); }
// Four row groups where a sequence's first keys pass many tiles of rows (their workgroup outlasts the launch: the bf16 case above 255 / 291 us
// with four / two), two of them and twice the workgroups a unit where they pass few (the f32 case 124 / 113, 8 sequences of up to 1000 192 / 174; the
// border is crude: the bf16 case with sequences of up to 512 takes 64 / 73); rows of 512 bytes leave room for two
int row_groups(const SeqArgs& f) {
  const long long turns = (long long)f.rows_q / f.batch * (f.heads / f.kv_heads) / 32;
  return (f.dtype == SEQ_F32 ? 4 : 2) * (f.dim <= 64 ? 64 : 128) <= 256 && turns >= 32 ? 4 : 2;
}

template <typename T, int DP, int RG, int KS> hipError_t grad_q(const SeqGradArgs& a, hipStream_t s) {
  static int done[kMaxDevices];
  constexpr int BN = RG == 4 ? 64 : 32, tiles_lds = KS * 4 * BN * SeqTile<T, DP>::kRow, join = (KS - 1) * RG * (DP / 32) * 16 * 256, lds = tiles_lds > join ? tiles_lds : join;
  static_assert(lds <= 160 * 1024, "LDS");
  opt_in_dynamic_lds((const void*)seq_dq_kernel<T, DP, RG, KS>, lds, done);
  const SeqArgs& f = a.f;
  const int tiles = (int)tiles_of(f.rows_q, f.batch, 32 * RG);
  vnr_launch(seq_dq_kernel<T, DP, RG, KS>, dim3((unsigned)tiles * f.heads), dim3(64 * RG * KS), lds, s, a, tiles);
  return hipGetLastError();
}
template <typename T, int DP, int KG, int HG> hipError_t grad_kv(const SeqGradArgs& a, hipStream_t s) {
  static int done[kMaxDevices];
  constexpr int tiles_lds = HG * 2 * (2 * 32 * SeqTile<T, DP>::kRow + (SeqTile<T, DP>::kRow > 256 ? 512 : 256)), join = (HG - 1) * KG * (DP / 32) * 16 * 256, lds = tiles_lds > join ? tiles_lds : join;
  static_assert(lds <= 160 * 1024, "LDS");
  opt_in_dynamic_lds((const void*)seq_dkv_kernel<T, DP, KG, HG>, lds, done);
  const SeqArgs& f = a.f;
  const int tiles = (int)tiles_of(f.rows_k, f.batch, 32 * KG);
  vnr_launch(seq_dkv_kernel<T, DP, KG, HG>, dim3((unsigned)tiles * f.kv_heads), dim3(64 * KG * HG), lds, s, a, tiles);
  return hipGetLastError();
}
template <typename T, int DP> hipError_t grad(const SeqGradArgs& a, int cus, hipStream_t s) {
  hipError_t e = hipSuccess;
  const SeqArgs& f = a.f;
  // 128 query rows a workgroup where that makes two for each compute unit, else 64 (32 utterances of up to 400 rows, 4 heads, f32: both kernels
  // 135 / 113 us with 128 / 64; 4 sequences of up to 512, 32 heads of 128, bf16: 78 / 73, of up to 2048: 256 / 269)
  const long long wgs = tiles_of(f.rows_q, f.batch, 128) * f.heads;
  if (f.rows_q > 0) e = wgs >= 2LL * cus ? grad_q<T, DP, 4, 1>(a, s) : grad_q<T, DP, 2, 2>(a, s);
  if (e != hipSuccess || f.rows_k == 0) return e;
  if (row_groups(f) == 4) return grad_kv<T, DP, 2, (sizeof(T) * DP > 256 ? 2 : 4)>(a, s);
  return grad_kv<T, DP, 2, 2>(a, s);
}
template <typename T> hipError_t grad(const SeqGradArgs& a, int cus, hipStream_t s) { return a.f.dim <= 64 ? grad<T, 64>(a, cus, s) : grad<T, 128>(a, cus, s); }
}  // namespace

// (256 threads a workgroup of dQ, of 128 rows at least where there are more than the chip holds; 64 keys and 128 threads a row group of dK and dV)
bool seq_grad_fits(const SeqArgs& f) {
  return tiles_of(f.rows_q, f.batch, 128) * f.heads < 1LL << 24 && tiles_of(f.rows_k, f.batch, 64) * f.kv_heads < (1LL << 32) / (128 * row_groups(f));
}
hipError_t launch_seq_grad(const SeqGradArgs& a, int cus, hipStream_t s) {
  if (a.f.dtype == SEQ_F32) return grad<float>(a, cus, s);
  if (a.f.dtype == SEQ_F16) return grad<_Float16>(a, cus, s);
  return grad<sq_bf16>(a, cus, s);
}
}  // namespace vnr
