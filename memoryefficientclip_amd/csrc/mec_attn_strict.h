// Attention of rows that do not see all of a tile, without products of what they do
// not see.
//
// A probability of 0 times an inf or a NaN is NaN: where a tile is seen in part
// (causal), a key's inf or NaN would pass on to rows that do not see it.  Rather than
// look at all values, the kernels look for a NaN in what they have in the end, and a
// wave that finds one does its work again here, row by row: 32 rows (or keys), one a
// lane as in the accumulators, against one key (or query) at a time, of those that are
// seen alone.  About 20 times the time of the tiles, for sequences with an inf or a NaN.
//
// Functions of their own, not inlined, whose results come back in memory: the kernels'
// registers are not theirs to take.
#pragma once
#include "mec_attn.h"

namespace mec {
namespace attn {

template <class O, int DB>
__device__ __forceinline__ bool any_nan(const f32x16 (&acc)[DB]) {
  bool nan = false;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) nan |= __builtin_isnan(acc[db][e]);
  return __any(nan);
}

// The tiles first, first + step, ... below last, of `size` rows each.
struct Range {
  int first, last, step, size;
};

// A lane's elements of a row, 32 db + 8 (i / 4) + 4 half + i % 4, and its part of a product of rows.
template <class T, int KS>
struct Line {
  static constexpr int DB = (KS + 1) / 2;
  static __device__ __forceinline__ float dot(const T* x, const T* y, bool valid, int half, int d) {
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      sum += Ops<T>::dot(Ops<T>::load_row(x, valid, s, half, d), Ops<T>::load_row(y, true, s, half, d));
    return sum + other_half(sum);
  }
  static __device__ __forceinline__ void add(float* acc, const T* x, int half, int d, float w, bool in) {
    if (!in) return;
    for (int i = 0; i < 4 * DB; ++i)
      for (int e = 0; e < 4; ++e) {
        const int at = 8 * i + 4 * half + e;
        if (at < d) acc[4 * i + e] = fmaf(w, value(x[at]), acc[4 * i + e]);
      }
  }
};

// o (16 DB values), m, l of k_attn_forward; a row sees the keys below `see`, none of the wave's those from `end` on.
template <class T, int KS>
__device__ __attribute__((noinline)) void strict_forward(const T* q, bool live, const T* k, int64_t k_pitch, const T* v,
                                                         int64_t v_pitch, int d, Range r, int end, int see, float c,
                                                         float* o) {
  const int half = (threadIdx.x >> 5) & 1;
  constexpr int N = 16 * ((KS + 1) / 2);
  float m = -kInf, l = 0.f;
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  for (int tile = r.first; tile < r.last; tile += r.step)
    for (int j = tile * r.size; j < min((tile + 1) * r.size, end); ++j) {
      const bool in = j < see;
      float x = Line<T, KS>::dot(q, k + j * k_pitch, live, half, d) * c;
      x = in ? x : -kInf;
      const float now = fmaxf(m, x), f = now == -kInf ? 1.f : fast_exp2(m - now);
      m = now;
      const float p = in ? fast_exp2(x - (now == -kInf ? 0.f : now) + Ops<T>::BIAS) : 0.f;
      l = l * f + (half ? 0.f : p);  // (the kernel adds the halves)
      for (int i = 0; i < N; ++i) o[i] *= f;
      Line<T, KS>::add(o, v + j * v_pitch, half, d, p, in);
    }
  o[N] = m;
  o[N + 1] = l;
}

// dq / scale of k_attn_dq.
template <class T, int KS>
__device__ __attribute__((noinline)) void strict_dq(const T* q, const T* g, bool live, const T* k, int64_t k_pitch,
                                                    const T* v, int64_t v_pitch, int d, Range r, int end, int see, float c,
                                                    float l2, float delta, float* acc) {
  const int half = (threadIdx.x >> 5) & 1;
  for (int i = 0; i < 16 * ((KS + 1) / 2); ++i) acc[i] = 0.f;
  for (int tile = r.first; tile < r.last; tile += r.step)
    for (int j = tile * r.size; j < min((tile + 1) * r.size, end); ++j) {
      const float x = Line<T, KS>::dot(q, k + j * k_pitch, live, half, d) * c;
      const float p = Line<T, KS>::dot(g, v + j * v_pitch, live, half, d);
      Line<T, KS>::add(acc, k + j * k_pitch, half, d, fast_exp2(x - l2) * (p - delta), j < see);
    }
}

// The queries of all heads of a key head, their gradients, lse and delta: `each` tiles of a head, from tile `skip` on.
template <class T>
struct Queries {
  const T *q, *g;
  int64_t q_pitch, q_head, g_pitch, g_head;
  const float *lse, *delta;  // a head's are `queries` apart
  int queries, nq, each, skip;
};
// dk / scale and dv / GRAD_UNIT of k_attn_dkv (16 DB values each); a key is seen by the queries from `seen` on.
template <class T, int KS>
__device__ __attribute__((noinline)) void strict_dkv(const T* k, const T* v, bool live, Queries<T> s, int d, Range r,
                                                     int seen, float c, float* acc) {
  const int half = (threadIdx.x >> 5) & 1;
  constexpr int N = 16 * ((KS + 1) / 2);
  for (int i = 0; i < 2 * N; ++i) acc[i] = 0.f;
  for (int tile = r.first; tile < r.last; tile += r.step) {
    const int h = tile / s.each, i0 = (s.skip + tile % s.each) * r.size;
    for (int i = i0; i < min(i0 + r.size, s.nq); ++i) {
      const T *q = s.q + h * s.q_head + i * s.q_pitch, *g = s.g + h * s.g_head + i * s.g_pitch;
      const float x = Line<T, KS>::dot(k, q, live, half, d) * c, p = Line<T, KS>::dot(v, g, live, half, d);
      const int64_t at = (int64_t)h * s.queries + i;
      const float w = fast_exp2(x - s.lse[at] + Ops<T>::GRAD_BIAS);
      Line<T, KS>::add(acc, q, half, d, w * (Ops<T>::GRAD_UNIT * (p - s.delta[at])), live && i >= seen);
      Line<T, KS>::add(acc + N, g, half, d, w, live && i >= seen);
    }
  }
}
template <int DB>
__device__ __forceinline__ void take(f32x16 (&acc)[DB], const float* from) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] = from[16 * db + e];
}

}  // namespace attn
}  // namespace mec
