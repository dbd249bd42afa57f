// New keys and values into a paged cache, turned by their positions on the way (and the queries of the same tokens beside them).
// Bound by memory: every element is read once and written once, 16 bytes a lane (32 in 32 bits): prompts of 17555 rows in all, 32 + 8 heads of
// 128, bf16: 84 us = 5.2 TB/s, as fast as a large copy; 8 rows 4.2 us, a launch and three loads that wait for each other (start, page, row).  One workgroup a token: the token's
// angles stay in registers while a thread goes over its share of the heads.
#include "sequence.h"

namespace vnr {
namespace {

template <typename T> struct Turn {
  typedef typename SeqVec<T>::v8 v8;
  // channels 8 u .. of the first half with those of the second: (a, b) -> (a cos - b sin, b cos + a sin), in 32 bits, rounded once
  static __device__ __forceinline__ void halves(v8& a, v8& b, const float (&cs)[8], const float (&sn)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (float)a[e], y = (float)b[e];
      a[e] = (T)__builtin_fmaf(x, cs[e], -(y * sn[e]));
      b[e] = (T)__builtin_fmaf(y, cs[e], x * sn[e]);
    }
  }
  // neighbouring channels of one chunk
  static __device__ __forceinline__ void pairs(v8& a, const float (&cs)[8], const float (&sn)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = (float)a[2 * e], y = (float)a[2 * e + 1];
      a[2 * e] = (T)__builtin_fmaf(x, cs[e], -(y * sn[e]));
      a[2 * e + 1] = (T)__builtin_fmaf(y, cs[e], x * sn[e]);
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(256) seq_append_kernel(const SeqAppendArgs a) {
  typedef typename SeqVec<T>::v8 v8;
  const int token = blockIdx.x;
  int start = 0;
  const int b = seq_owner(a.cu, a.batch, a.rows, token, start);
  if (b < 0) return;                                         // a row outside the sequences: nothing is read or written
  int pos = a.ctx[b];
  pos = (pos < 0 ? 0 : pos);
  const long long room = (long long)a.table_width << a.page_shift, p64 = (long long)pos + (token - start);
  if (p64 >= room) return;                                   // behind the table's end there is no place, and no angle
  pos = (int)p64;
  const int page = a.table[(size_t)b * a.table_width + (pos >> a.page_shift)];
  const bool held = (unsigned)page < (unsigned)a.pages;      // a page that is none: K and V are dropped, the query is turned all the same
  const long long slot = pos & ((1 << a.page_shift) - 1);

  const int D = a.dim, half = a.rot_dim >> 1;
  const int turning = a.interleaved ? a.rot_dim >> 3 : half >> 3;          // items that turn (a pair of chunks, or one chunk of pairs)
  const int items = turning + ((D - a.rot_dim) >> 3);
  const int u = threadIdx.x % items, h0 = threadIdx.x / items, slots = 256 / items;
  if (h0 >= slots) return;
  const bool turns = u < turning;
  const int at = turns ? 8 * u : a.rot_dim + 8 * (u - turning);            // first channel of the item (its second chunk: + half)
  float cs[8], sn[8];
  if (turns) {
    const float* r = a.rotation + (size_t)pos * a.rot_dim + (a.interleaved ? 4 * u : 8 * u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool ok = !a.interleaved || e < 4;
      cs[e] = ok ? r[e] : 1.f; sn[e] = ok ? r[half + e] : 0.f;
    }
  }
  const bool two = turns && !a.interleaved;
  auto place = [&](int head) { return (((long long)page * a.kv_heads + head) << a.page_shift) * D + slot * D; };
  const int nq = a.q ? a.heads : 0, all = a.kv_heads + nq;
  for (int h = h0; h < all; h += slots) {                    // keys, then queries
    const bool key = h < a.kv_heads;
    if (key && !held) continue;
    const T* src = key ? (const T*)a.k + token * a.ldk + (long long)h * D : (const T*)a.q + token * a.ldq + (long long)(h - a.kv_heads) * D;
    T* dst = key ? (T*)a.kc + place(h) : (T*)a.q_out + token * a.ldqo + (long long)(h - a.kv_heads) * D;
    v8 x = *reinterpret_cast<const v8*>(src + at);
    if (two) {
      v8 y = *reinterpret_cast<const v8*>(src + at + half);
      Turn<T>::halves(x, y, cs, sn);
      *reinterpret_cast<v8*>(dst + at) = x;
      *reinterpret_cast<v8*>(dst + at + half) = y;
    } else {
      if (turns) Turn<T>::pairs(x, cs, sn);
      *reinterpret_cast<v8*>(dst + at) = x;
    }
  }
  if (!held) return;
  for (int h = h0; h < a.kv_heads; h += slots) {             // values: as they are
    const T* src = (const T*)a.v + token * a.ldv + (long long)h * D;
    T* dst = (T*)a.vc + place(h);
    *reinterpret_cast<v8*>(dst + at) = *reinterpret_cast<const v8*>(src + at);
    if (two) *reinterpret_cast<v8*>(dst + at + half) = *reinterpret_cast<const v8*>(src + at + half);
  }
}

// cosines | sines of position / base^(2 i / rot_dim), from 64 bits: an angle of position 100000 keeps its last digits
__global__ void __launch_bounds__(256) rotation_table_kernel(int positions, int half, double log_base, float* out) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)positions * half) return;
  const int p = (int)(i / half), c = (int)(i - (long long)p * half);
  const double x = (double)p * exp(-log_base * (double)c / (double)half);
  out[(long long)p * 2 * half + c] = (float)cos(x);
  out[(long long)p * 2 * half + half + c] = (float)sin(x);
}
}  // namespace

hipError_t launch_seq_append(const SeqAppendArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.dtype == SEQ_F32) vnr_launch(seq_append_kernel<float>, dim3(a.rows), dim3(256), 0, s, a);
  else if (a.dtype == SEQ_F16) vnr_launch(seq_append_kernel<_Float16>, dim3(a.rows), dim3(256), 0, s, a);
  else vnr_launch(seq_append_kernel<sq_bf16>, dim3(a.rows), dim3(256), 0, s, a);
  return hipGetLastError();
}
hipError_t launch_rotation_table(int positions, int rot_dim, double base, float* out, hipStream_t s) {
  const long long n = (long long)positions * (rot_dim / 2);
  if (n <= 0) return hipSuccess;
  vnr_launch(rotation_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, positions, rot_dim / 2, log(base), out);
  return hipGetLastError();
}
}  // namespace vnr
