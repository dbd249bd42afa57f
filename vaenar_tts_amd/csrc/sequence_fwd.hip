// Attention forward on packed sequences and over a paged cache: out = softmax(scale q k' + mask) v, one pass over the keys with the running
// maximum and sum of every row.
//
//   S' = K Q'   (keys along the product's rows, the 32 query rows of a tile along its columns: a lane owns ONE query row, its maximum and
//               sum are register arithmetic plus one exchange with the lane 32 away)
//   P  = exp2(c S - c m), c = scale log2 e; m is a running bound of the row: it moves only when a tile exceeds it by more than 8 / c, so that
//        the accumulators are rarely rescaled (in float16 by more than 4 / c, see Weight).  P is rounded to the operands' type (by at most 2^-8 of its
//        value, in float16 2^-11 of it or 2^-36 of the row's largest; nothing in 32 bits) for the second product, as the values of V are; where memory
//        or latency bounds the launch (over a cache with up to 64 rows, packed with 32) what that rounding left goes through a second product.  The
//        row sums take the unrounded values, in 32 bits
//   O' += V' P'  with P' straight out of the first product's registers (sequence.h: seq_col's key order)
//
// K and V tiles come straight from memory to LDS (16 bytes a lane, no registers), the next tile while this one is multiplied.
//
// What bounds it: long prompts the matrix pipe and the exponentials between its products (4 prompts of up to 4096 rows, 32 heads of 128, bf16, causal:
// 412 - 425 us by card = 0.96 - 0.93 PFLOP/s of the products that are not masked; 851 thousand cycles, 45 % of which the pipe is busy; the waves wait
// 21 % of theirs for tiles and barriers and 35 % for each other's turns on the units); a decoding step memory (64 sequences of up to 4096 keys, 32
// heads over 8 of 128, bf16: 117 us = 4.8 TB/s, 2 of 100000 keys 140 us = 5.5; a large copy reaches 5.0); few short sequences the way through one
// workgroup (4 utterances of up to 101 rows: 10 us; the append of 8 rows, three loads that wait for each other and one store, takes 4.2).
#include "sequence.h"

namespace vnr {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
// How far (log2) a row may exceed its running bound before it is moved, and the power of two that its weights carry.  float16 has no weights of its own
// precision below 2^-14 and none below 2^-25: there they are 2^11 times what they are elsewhere (at most 2^15 with the slack of the bound), so that those
// down to 2^-25 of the largest are rounded like any other and what is lost of the rest is 2^-36 of it.
template <typename T> struct Weight { static constexpr float kSlack = __is_same(T, _Float16) ? 4.f : 8.f, kLift = __is_same(T, _Float16) ? 11.f : 0.f, kTimes = __is_same(T, _Float16) ? 2048.f : 1.f; };
constexpr int kMaxSplits = 64;

// Where the rows of a task's keys and values are.  `n`: keys of the sequence; rows from n on read as zeros.  A whole tile goes by scalar
// addresses (a transfer's rows lie in one page); the last tile of a sequence, heads narrower than the tile and pages of fewer rows than a
// transfer go by an address in every lane, which points to zeros where there is nothing.
template <typename T, int DP, bool PAGED, int N>
struct KeySource {
  typedef SeqTile<T, DP> L;
  static constexpr int kRowsOf = SeqLanes<T, DP>::kRowsOf;
  const char *k, *v; long long ldk, ldv;                     // bytes from a row to the next (paged: of a page)
  const int32_t* table; int last, shift, pages, kv_heads, head, dim, n; const void* zero;
  bool plain;                                                // whole tiles may go by scalar addresses
  SeqLanes<T, DP> wk, wv;
  int page[N];                                               // of the transfers of the tile to come
  __device__ __forceinline__ void look(int k0, int first) {
    if constexpr (PAGED) {
      if (!plain) return;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int x = (k0 + (first + i) * kRowsOf) >> shift;
        page[i] = seq_scalar(table + (x < last ? x : last));
      }
    }
  }
  // transfers first .. first + N - 1 of the tile of `rows` keys that starts at key k0; tk, tv: where its K and V lie in LDS
  __device__ __forceinline__ void fetch(int k0, int rows, int first, unsigned tk, unsigned tv, int lane) const {
    if (plain && k0 + rows <= n) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = k0 + (first + i) * kRowsOf;
        const char *pk, *pv;
        bool there = true;
        if constexpr (PAGED) {
          const long long o = ((((long long)page[i] * kv_heads + head) << shift) + (row & ((1 << shift) - 1))) * ldk;
          pk = k + o; pv = v + o;
          there = (unsigned)page[i] < (unsigned)pages;
        } else {
          pk = k + row * ldk; pv = v + row * ldv;
        }
        if (!there) { pk = pv = (const char*)zero; }
        seq_dma16(pk, there ? wk.at(i) : 0u, tk + (first + i) * 1024);
        seq_dma16(pv, there ? (PAGED ? wk : wv).at(i) : 0u, tv + (first + i) * 1024);
      }
      return;
    }
    asm volatile("" : "+v"(lane));                           // (opaque: or what follows from it is kept in registers all the way)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (first + i) * kRowsOf + lane / L::kChunks, c = (lane % L::kChunks) ^ L::turn(r), row = k0 + r;
      bool ok = row < n && c * L::kPer < dim;
      const char *pk, *pv;                                   // (addresses only: where `ok` is false nothing reads there)
      if constexpr (PAGED) {
        const int x = row >> shift, pg = table[x < last ? x : last];
        const long long o = ((((long long)pg * kv_heads + head) << shift) + (row & ((1 << shift) - 1))) * ldk + c * 16;
        pk = k + o; pv = v + o;
        ok = ok && (unsigned)pg < (unsigned)pages;
      } else {
        pk = k + row * ldk + c * 16; pv = v + row * ldv + c * 16;
      }
      seq_dma16(ok ? (const void*)pk : zero, tk + (first + i) * 1024);
      seq_dma16(ok ? (const void*)pv : zero, tv + (first + i) * 1024);
    }
  }
};

// One workgroup: four waves, RG of them side by side along the rows (32 each) and KS along the keys.  The waves of one key group read the same
// tiles of BN keys; the groups take tiles in turn and their results for the same rows are joined through LDS at the end.  4 x 1 reads every
// key tile once for 128 rows (long prompts, long chunks), 2 x 2 has 64 rows (a decoding step), 1 x 4 has 32 and no barrier in its loop.
template <typename T, int DP, int RG, int KS>
struct Fwd {
  typedef SeqTile<T, DP> L;
  typedef typename SeqVec<T>::v8 v8;
  static constexpr int BN = RG == 4 ? 64 : 32, NJ = BN / 32, BM = 32 * RG;
  static constexpr int kTile = BN * L::kRow;                 // bytes of one K or V tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kLds = 2 * KS * kStage + (3 * DP + 1) * 4;               // a tile that is read and one on its way; more of them cost more in workgroups a unit than they hide (16 ragged f16: 20 -> 27 us)
  static constexpr int kIssue = kTile / 1024 / RG;           // transfers of a wave for one tile of K (as many for V)
  static constexpr int kRegs = (DP / 32) * 16;               // accumulators of a lane
  static constexpr int kJoin = (KS - 1) * RG * (kRegs + 2) * 256;
  static_assert(kJoin <= 2 * KS * kStage, "the join lies where the tiles were");
};

// A row's weights under the bound m: exp2((s - sub) c + off).  What is taken off is the bound in units of log2, rounded once and the same wherever
// it is used, so that weights of different tiles stay in proportion.  Beyond 2^16 that rounding is more than the weights can bear (from 2^27 on they
// would be infinite or nothing), and logits and bound are subtracted in front of the product instead.
struct Base { float sub, off; };
template <typename T> __device__ __forceinline__ Base base_of(float m, float c) {
#pragma clang fp contract(off)
  const float off = Weight<T>::kLift - m * c;
  const bool far = __builtin_fabsf(off) > 65536.f, none = m == -__builtin_inff();
  const Base b = {far && !none ? m : 0.f, none ? 0.f : (far ? Weight<T>::kLift : off)};
  return b;
}
// weights under one base over those under another
__device__ __forceinline__ float ratio(const Base& to, const Base& from, float c) { return __builtin_amdgcn_exp2f(__builtin_fmaf(from.sub - to.sub, c, to.off - from.off)); }
// the logarithm of a row's sum `l` of weights: what the base's rounding left belongs to it
template <typename T> __device__ __forceinline__ float log_sum(float m, float l, float scale) {
  const float c = scale * kLog2e;
  const Base b = base_of<T>(m, c);
  return m * scale + (__logf(l * (1.f / Weight<T>::kTimes)) - kLn2 * __builtin_fmaf(m - b.sub, c, b.off - Weight<T>::kLift));
}

// The pieces of a row's keys joined by one wave, lanes along the channels
template <typename T>
__device__ __forceinline__ void join_row(const SeqArgs& a, long long pr, long long n, int token, int head, int lane) {
  float m = -__builtin_inff(), l = 0.f;
  if (lane < a.splits) { const sq_f2 x = *reinterpret_cast<const sq_f2*>(a.ml + 2 * (lane * n + pr)); m = x[0]; l = x[1]; }
  constexpr int N = 16;
  const int col = 2 * lane < a.dim ? 2 * lane : 0;
  sq_f2 x = {0.f, 0.f};
  float f = 0.f, sum = 0.f, top = 0.f;
  for (int s0 = 0; s0 < a.splits; s0 += N) {
    sq_f2 p[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {                            // (on their way before the weights are known; behind the last piece: the last one again)
      const int s = s0 + i < a.splits ? s0 + i : a.splits - 1;
      p[i] = *reinterpret_cast<const sq_f2*>(a.part + (s * n + pr) * a.dim + col);
    }
    if (s0 == 0) {
      if (l == 0.f) m = -__builtin_inff();
      top = m;
#pragma unroll
      for (int s = 32; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
      const float c = a.scale * kLog2e;
      f = l != 0.f ? ratio(base_of<T>(top, c), base_of<T>(m, c), c) : 0.f;
      sum = l * f;
#pragma unroll
      for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s, 64);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = s0 + i;
      const float fs = __shfl(f, s & 63, 64);
      if (s < a.splits && fs != 0.f) { x[0] += fs * p[i][0]; x[1] += fs * p[i][1]; }      // (an empty piece has left nothing)
    }
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  if (2 * lane < a.dim) {
    T* op = (T*)a.out + token * a.ldo + (long long)head * a.dim + col;
    op[0] = (T)(x[0] * inv); op[1] = (T)(x[1] * inv);
  }
  if (a.lse && lane == 0) a.lse[(long long)head * a.rows_q + token] = sum != 0.f ? log_sum<T>(top, sum, a.scale) : -__builtin_inff();
}

template <typename T, int DP, bool PAGED, int RG, int KS>
__global__ void __launch_bounds__(64 * RG * KS, sizeof(T) == 2 ? 2 : 1)
seq_fwd_kernel(const SeqArgs a, const int tiles) {
  typedef Fwd<T, DP, RG, KS> F;
  typedef SeqTile<T, DP> L;
  typedef typename F::v8 v8;
  extern __shared__ __attribute__((aligned(512))) char smem[];         // (SeqReads: tiles start at multiples of their row)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % RG, kg = wave / RG;
  const int l31 = lane & 31, g = lane >> 5;

  // ---- which rows: packed: one query head, rows = tokens; paged: the heads of a group side by side, rows = (token, head) ------------------------
  const int group = a.heads / a.kv_heads;
  const int mult = PAGED ? group : 1;
  int task = seq_task(blockIdx.x, gridDim.x);
  int kvh, hq, split = 0;
  if (PAGED) { split = task % a.splits; task /= a.splits; hq = 0; kvh = task / tiles; task -= kvh * tiles; }
  else { hq = task % group; task /= group; kvh = task / tiles; task -= kvh * tiles; }
  SeqWhere w;
  if (!seq_find(a.cu_q, a.batch, a.rows_q, mult, F::BM, task, PAGED ? a.ctx : a.cu_k, PAGED ? 0 : 1, w)) return;
  const int rows = w.n * mult, r0 = ((rows + F::BM - 1) / F::BM - 1 - w.tile) * F::BM;            // (from the sequence's end: its last rows see most keys)
  int nk, ahead, kstart = 0;                                 // keys of the sequence; keys in front of its first new row
  if (PAGED) {
    ahead = w.x0 < 0 ? 0 : (w.x0 > a.max_context ? a.max_context : w.x0);
    const long long room = (long long)a.table_width << a.page_shift;
    nk = ahead + w.n;
    nk = nk > a.max_context ? a.max_context : nk;
    nk = nk > room ? (int)room : nk;
  } else {
    seq_clamp(w.x0, w.x1, a.rows_k, kstart, nk);
    ahead = nk - w.n;
  }
  const int row = r0 + 32 * rg + l31;                        // this lane's row; both halves of the wave have the same 32
  const bool live = row < rows;
  const int token = w.start + (live ? row / mult : 0), head = kvh * group + (PAGED ? row % mult : hq);
  int limit = 0;                                             // keys this row sees: 0 .. limit - 1
  if (live) { limit = (PAGED || a.causal) ? ahead + row / mult + 1 : nk; limit = limit < 0 ? 0 : (limit > nk ? nk : limit); }
  // the same for the first and the last row of the workgroup and of the wave: tiles behind `some` are not looked at, tiles in
  // front of `all` need no mask
  auto seen = [&](int r) { const int x = (PAGED || a.causal) ? ahead + r / mult + 1 : nk; return x < 0 ? 0 : (x > nk ? nk : x); };
  const int last = (r0 + F::BM < rows ? r0 + F::BM : rows) - 1;
  const int wfirst = r0 + 32 * rg, wlast = (wfirst + 32 < rows ? wfirst + 32 : rows) - 1;
  const int some = seen(last);
  const int wall = wfirst < rows ? seen(wfirst) : nk, wsome = wfirst < rows ? seen(wlast) : 0;
  int k_begin = 0, k_end = some;
  if (PAGED && a.splits > 1) { k_begin = split * a.chunk; k_end = k_begin + a.chunk < some ? k_begin + a.chunk : some; }

  KeySource<T, DP, PAGED, F::kIssue> src;
  constexpr int es = sizeof(T);
  if (PAGED) {
    src.k = (const char*)a.k; src.v = (const char*)a.v; src.ldk = src.ldv = (long long)a.dim * es;
    src.table = a.table + (size_t)w.b * a.table_width; src.last = a.table_width - 1; src.shift = a.page_shift; src.pages = a.pages;
    src.plain = a.dim == DP && (1 << a.page_shift) >= src.kRowsOf;
  } else {
    src.k = (const char*)a.k + (kstart * a.ldk + (long long)kvh * a.dim) * es; src.v = (const char*)a.v + (kstart * a.ldv + (long long)kvh * a.dim) * es;
    src.ldk = a.ldk * es; src.ldv = a.ldv * es;
    src.plain = a.dim == DP && a.ldk < (1 << 24) && a.ldv < (1 << 24) && !(src.ldk % L::kRow) && !(src.ldv % L::kRow);         // (SeqLanes; a lane's offset in 32 bits)
  }
  src.kv_heads = a.kv_heads; src.head = kvh; src.dim = a.dim; src.n = nk; src.zero = a.zero;
  src.wk.set((unsigned)src.ldk, lane, rg * F::kIssue);
  if (!PAGED) src.wv.set((unsigned)src.ldv, lane, rg * F::kIssue);

  v8 qf[DP / 16];
  {
    const T* qp = (const T*)a.q + token * a.ldq + (long long)head * a.dim;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) qf[t] = seq_load8<T>(qp + 16 * t + 8 * g, live && 16 * t + 8 * g < a.dim, a.zero);
  }
  f32x16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -__builtin_inff(), l = 0.f;                      // running bound (of the raw products) and this lane's part of the row sum
  const float c = a.scale * kLog2e;
  Base w0 = {0.f, 0.f};                                      // base_of(m, c)
  bool far = false;                                          // is any lane's beyond 2^16? (the same for the wave)

  char* base = smem + kg * 2 * F::kStage;
  const unsigned lds = seq_lds(base);
  constexpr int step = F::BN * KS;
  // ---- one tile: the logits of its keys, their weights, their share of the result -----------------------------------------------------
  f32x16 s[F::NJ];
  SeqReads<T, DP> reads;
  reads.set(lane);
  auto logits = [&](unsigned tk) {
    const unsigned at = seq_at(tk, reads.row);
#pragma unroll
    for (int j = 0; j < F::NJ; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[j][i] = 0.f;
    constexpr int n = DP / 16;
    seq_run<T, F::NJ * n>([&](int i) { return seq_row<T, DP>(at, 32 * (i / n), i % n); }, [&](int i, const v8& k) { s[i / n] = seq_mma(k, qf[i % n], s[i / n]); });
  };
  auto weights = [&](int k0) {
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
    if (__builtin_amdgcn_ballot_w64((mx - m) * c > Weight<T>::kSlack || (mx > m && m == -__builtin_inff()))) {
      const float m1 = fmaxf(m, mx);
      const Base b = base_of<T>(m1, c);
      const float f = m == -__builtin_inff() ? 0.f : ratio(b, w0, c);
      m = m1; w0 = b;
      far = __builtin_amdgcn_ballot_w64(b.sub != 0.f) != 0;
      l *= f;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= f;
    }
    if (far) {
#pragma unroll
      for (int j = 0; j < F::NJ; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[j][i] -= w0.sub;
    }
#pragma unroll
    for (int j = 0; j < F::NJ; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) { s[j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], c, w0.off)); l += s[j][i]; }
  };
  auto result = [&](unsigned tv) {
    const unsigned at = seq_at(tv, reads.col);
    constexpr int n = DP / 32;
    constexpr bool fine = sizeof(T) == 2 && (PAGED ? RG < 4 : RG == 1);      // (memory or latency bounds these: the second half of the weights is free)
    v8 p, rest;
    seq_run<T, F::NJ * 2 * n>([&](int i) { return seq_col<T, DP>(at, 16 * (i / n), i % n); },
                              [&](int i, const v8& v) {
                                if (i % n == 0) {
                                  if constexpr (fine) p = seq_pack<T>(s[i / n / 2], i / n % 2, rest); else p = seq_pack<T>(s[i / n / 2], i / n % 2);
                                }
                                o[i % n] = seq_mma(v, p, o[i % n]);
                                if constexpr (fine) o[i % n] = seq_mma(v, rest, o[i % n]);
                              });
  };
  const int mine = rg * F::kIssue;                           // this wave's first transfer of a tile
  // The first turn of the loop only fetches (one place in the code for it: short launches wait for their instructions, too).  Key groups go
  // through the loop equally often: its barrier is everybody's.
  seq_settle(qf);
  int *what = reinterpret_cast<int*>(smem + 2 * KS * F::kStage), *flag = what + 3 * DP;         // seq_apart's, and the last tiles that needed it
  for (int i = threadIdx.x; i < 3 * DP; i += 64 * RG * KS) what[i] = 0x7fffffff;
  if (threadIdx.x == 0) *flag = -1;
  if (RG == 1) __syncthreads();
  const int all = seen(r0);                                  // what the workgroup's first row sees
  int stage = 0, k0 = k_begin + (kg - KS) * F::BN;
  src.look(k0 + step, mine);
  for (int kt = k_begin - step; kt < k_end; kt += step, k0 += step, stage ^= F::kStage) {
    seq_dma_wait();
    if (RG > 1) __syncthreads();                             // this tile is there, and nobody reads the other stage any more
    if (k0 + step < k_end) {
      const unsigned t = lds + (stage ^ F::kStage);
      src.fetch(k0 + step, F::BN, mine, t, t + F::kTile, lane);
      src.look(k0 + 2 * step, mine);
    }
    if (kt < k_begin) continue;
    // Where the diagonal runs through the tiles -- keys that are there and that some row does not see --: is any value in them not finite?
    if (kt + step > all && all < nk) {
      int me = rg * 64 + lane;                               // (an opaque copy: or the addresses below are kept in registers all the way)
      asm volatile("" : "+v"(me));
      if (k0 < k_end && seq_tainted<T, DP, F::BN>(base + stage + F::kTile, me, 64 * RG) && lane == 0) *flag = kt;
      __syncthreads();
      if (*flag == kt) {
        if (k0 < k_end) seq_apart<T, DP, F::BN>(base + stage + F::kTile, what, k0, me, 64 * RG);
        __syncthreads();
      }
    }
    if (k0 >= k_end || k0 >= wsome) continue;
    logits(lds + stage);
    weights(k0);
    result(lds + stage + F::kTile);
  }
  l = seq_pair_sum(l);

  __syncthreads();
  const bool apart = *flag >= 0;                             // (in front of the join, which uses the tiles' place)
  if (KS > 1) {                                              // the key groups' parts of the same rows: the first group collects them
    float* x = reinterpret_cast<float*>(smem) + lane;        // [KS - 1][RG][registers, m, l][64]
    constexpr int N = F::kRegs;
    if (kg > 0) {
      float* y = x + ((kg - 1) * RG + rg) * (N + 2) * 64;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) y[(16 * d + i) * 64] = o[d][i];
      y[N * 64] = m; y[(N + 1) * 64] = l;
    }
    __syncthreads();
    for (int k = 0; kg == 0 && k < KS - 1; ++k) {
      const float* y = x + (k * RG + rg) * (N + 2) * 64;
      const float m2 = y[N * 64], l2 = y[(N + 1) * 64], m1 = fmaxf(m, m2);
      const Base b = base_of<T>(m1, c);
      const float f1 = m == -__builtin_inff() ? 0.f : ratio(b, base_of<T>(m, c), c), f2 = m2 == -__builtin_inff() ? 0.f : ratio(b, base_of<T>(m2, c), c);
      m = m1; l = l * f1 + l2 * f2;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * f1 + y[(16 * d + i) * 64] * f2;
    }
  }
  if (apart) {
    int half = g;
    asm volatile("" : "+v"(half));
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        typedef int i4 __attribute__((ext_vector_type(4)));
        const i4* w = reinterpret_cast<const i4*>(what + 32 * d + 8 * (i >> 2) + 4 * half);
        const i4 up = w[0], down = w[DP / 4], none = w[DP / 2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (up[e] < limit) o[d][i + e] += __builtin_inff();
          if (down[e] < limit) o[d][i + e] -= __builtin_inff();
          if (none[e] < limit) o[d][i + e] = __builtin_nanf("");
        }
        asm volatile("" ::: "memory");                       // (four channels at a time: this is rare, registers are not)
      }
  }
  if (PAGED && a.splits > 1) {
    const long long n = (long long)a.rows_q * a.heads;
    if (live && kg == 0) {
      const long long pr = split * n + (long long)token * a.heads + head;
      if (g == 0) { const sq_f2 x = {m, l}; *reinterpret_cast<sq_f2*>(a.ml + 2 * pr) = x; }
      float* op = a.part + pr * a.dim;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int col = 32 * d + 8 * (i >> 2) + 4 * g;
          if (col < a.dim && l != 0.f) seq_store4<float>(op + col, o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
        }
    }
    return;                                                  // (seq_join_kernel follows)
  }
  if (!live || kg > 0) return;
  const float inv = l != 0.f ? 1.f / l : 0.f;                // a row that sees nothing: zeros, and minus infinity for its sum
  T* op = (T*)a.out + token * a.ldo + (long long)head * a.dim;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int col = 32 * d + 8 * (i >> 2) + 4 * g;
      if (col < a.dim) seq_store4<T>(op + col, o[d][i] * inv, o[d][i + 1] * inv, o[d][i + 2] * inv, o[d][i + 3] * inv);
    }
  if (a.lse && g == 0) a.lse[(long long)head * a.rows_q + token] = l != 0.f ? log_sum<T>(m, l, a.scale) : -__builtin_inff();
}

template <typename T>
__global__ void __launch_bounds__(256) seq_join_kernel(const SeqArgs a) {
  const long long pr = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), n = (long long)a.rows_q * a.heads;
  if (pr >= n) return;
  const int token = (int)(pr / a.heads), head = (int)(pr - (long long)token * a.heads);
  int start;
  if (seq_owner(a.cu_q, a.batch, a.rows_q, token, start) < 0) return;          // rows outside the sequences stay as they were
  join_row<T>(a, pr, n, token, head, threadIdx.x & 63);
}

long long tiles_of(const SeqArgs& a, int mult, int bm) {     // at most: every sequence ends inside a tile
  return (long long)a.rows_q * mult / bm + (a.batch < a.rows_q ? a.batch : a.rows_q);
}
// workgroups of `row_waves` x 32 rows, and of four waves at most
long long grid_of(const SeqArgs& a, int row_waves, int splits) {
  return a.table ? tiles_of(a, a.heads / a.kv_heads, 32 * row_waves) * a.kv_heads * splits : tiles_of(a, 1, 32 * row_waves) * a.heads;
}
constexpr long long kMostWorkgroups = (1 << 24) - 1;         // of 256 threads

template <typename T, int DP, bool PAGED, int RG, int KS>
hipError_t fwd(const SeqArgs& a, hipStream_t s) {
  typedef Fwd<T, DP, RG, KS> F;
  static int done[kMaxDevices];
  constexpr int lds = F::kLds > F::kJoin ? F::kLds : F::kJoin;
  static_assert(lds <= 160 * 1024, "LDS");
  opt_in_dynamic_lds((const void*)seq_fwd_kernel<T, DP, PAGED, RG, KS>, lds, done);
  const int tiles = (int)tiles_of(a, PAGED ? a.heads / a.kv_heads : 1, F::BM);
  vnr_launch(seq_fwd_kernel<T, DP, PAGED, RG, KS>, dim3((unsigned)grid_of(a, RG, a.splits)), dim3(64 * RG * KS), lds, s, a, tiles);
  return hipGetLastError();
}
template <typename T, int DP, bool PAGED>
hipError_t fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s) {
  if (p.row_waves == 4) return fwd<T, DP, PAGED, 4, 1>(a, s);
  if (PAGED || p.row_waves == 2) return fwd<T, DP, PAGED, 2, 2>(a, s);
  return fwd<T, DP, false, 1, (sizeof(T) * DP > 256 ? 2 : 4)>(a, s);         // (rows of 512 bytes: two key groups fill the LDS)
}
template <typename T> hipError_t fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s) {
  if (a.dim <= 64) return a.table ? fwd<T, 64, true>(a, p, s) : fwd<T, 64, false>(a, p, s);
  return a.table ? fwd<T, 128, true>(a, p, s) : fwd<T, 128, false>(a, p, s);
}
long long join_grid(const SeqArgs& a) { return ((long long)a.rows_q * a.heads + 3) / 4; }
}  // namespace

// Rows a workgroup.  Packed: 128 (every key tile is read once for them) where that makes two workgroups for each compute unit; else 64, else 32
// with all four waves along the keys: a launch of few workgroups lasts as long as one of them (4 utterances of up to 101 rows, 4 heads, f32:
// 15.8 / 11.1 / 9.8 us with 128 / 64 / 32 rows; 16 of up to 800, f16: 20.2 / 18.6 / 26.2; 4 prompts of up to 4096, 32 heads of 128, bf16:
// 417 / 514 / 1138).  With the border at one workgroup for each unit, two and four: 32 utterances of up to 400, f32, 51.5 / 39.5 / 60.7; the 16,
// 19.8 / 18.8 / 27.0; prompts of up to 400, bf16, 16.2 / 17.5 / 44.0.  Over a cache: 64 rows where no sequence has more (group x new rows), else 128
// (one row for each of 64 sequences: 117.6 / 119.0 us with 64 / 128; chunks of up to 512: 250 / 182), and the keys are cut where the tiles alone leave
// compute units idle: two workgroups for each of them (4 rows over 4096 keys: 22.5 us with one, 18.1 with two, 17.9 with four; 2 over 100000: 149 /
// 143.5 / 150; chunks of 5 over 2000: 16.6 / 15.1 / 15.8), no piece shorter than 256 keys (1 row over 4096: 18.6 with 512, 15.3 with 256, 14.5 with
// 128, over 1000 14.7 / 11.4 / 9.9; chunks of 5 16.5 / 15.1 / 15.2) and at most 64 pieces, one a lane of the join (1 row of one cache head over
// 100000: 42.3 us, 67.8 with 32).
SeqPlan seq_plan(const SeqArgs& a, int cus) {
  SeqPlan p;
  const int group = a.heads / a.kv_heads;
  if (!a.table) {
    while (p.row_waves > 1 && grid_of(a, p.row_waves, 1) < 2LL * cus) p.row_waves /= 2;
    return p;
  }
  p.row_waves = (long long)a.max_new * group > 64 ? 4 : 2;
  const long long wgs = grid_of(a, p.row_waves, 1);
  long long want = wgs > 0 ? (2LL * cus + wgs - 1) / wgs : 1;
  const long long most = (a.max_context + 255) / 256;
  if (want > most) want = most;
  if (want > kMaxSplits) want = kMaxSplits;
  if (want < 1) want = 1;
  p.chunk = (int)(((a.max_context + want - 1) / want + 127) / 128 * 128);      // (whole tiles of every key group)
  p.splits = (a.max_context + p.chunk - 1) / p.chunk;
  return p;
}

bool seq_fwd_fits(const SeqArgs& a, const SeqPlan& p) {
  return grid_of(a, p.row_waves, p.splits) <= kMostWorkgroups && (p.splits == 1 || join_grid(a) <= kMostWorkgroups);
}
hipError_t launch_seq_fwd(const SeqArgs& a, const SeqPlan& p, hipStream_t s) {
  if (a.dtype == SEQ_F32) return fwd<float>(a, p, s);
  if (a.dtype == SEQ_F16) return fwd<_Float16>(a, p, s);
  return fwd<sq_bf16>(a, p, s);
}
hipError_t launch_seq_join(const SeqArgs& a, hipStream_t s) {
  const long long grid = join_grid(a);
  if (a.dtype == SEQ_F32) vnr_launch(seq_join_kernel<float>, dim3((unsigned)grid), dim3(256), 0, s, a);
  else if (a.dtype == SEQ_F16) vnr_launch(seq_join_kernel<_Float16>, dim3((unsigned)grid), dim3(256), 0, s, a);
  else vnr_launch(seq_join_kernel<sq_bf16>, dim3((unsigned)grid), dim3(256), 0, s, a);
  return hipGetLastError();
}
}  // namespace vnr
