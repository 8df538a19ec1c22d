// Rotation of queries and keys by positions on several axes, with the norm of
// each head in the same pass, and the gradient.
//
// A head x of d features is d / 2 pairs (a, b): (x[p], x[p + d/2]), or
// (x[2p], x[2p + 1]) interleaved.  Pair p belongs to one axis, and is turned by
// t = position[axis] * f(p), f(p) = theta^(-j / n) for the j-th of the axis's n
// pairs:
//   n = r w x, r = 1 / sqrt(mean x^2 + eps)    (n = x without a norm)
//   y = (a cos t - b sin t, b cos t + a sin t) of n's pairs
// and backwards, the turn being orthogonal,
//   g = dy turned by -t;  dw = sum over heads of g r x;
//   h = g w;  dx = r (h - (r x) mean(h r x)).
// The angle is formed in 64 bits and reduced to a part of a turn there: in 32
// bits the angle of position 10^6 is off by up to 0.03.
//
// Bound by memory: x is read and y written once (backwards dy and x read, dx
// written), all else is registers.  A wave takes a token's query heads, or its key
// heads: all of them, so that the angles are formed once, one pair a lane, and
// handed to the lanes that need them through LDS; one side, so that a lane holds
// the weights, and the sums of their gradients, of one.  In a head's row a
// lane holds VP pairs, both halves of each, so that the turn crosses no lanes;
// a group of 2^lg lanes is a row, and only the norm's sum of squares crosses
// them.  The next rows are on their way while the ones before are turned.
#pragma once
#include "mec_vec.h"

namespace mec {

constexpr int kRotaryWaves = 4;
constexpr int kMaxAxes = 8;
constexpr int kMaxHalf = 128;  // pairs of a head

struct RotaryShape {
  int64_t rows;       // batch * tokens
  int tokens;
  int heads[2];       // of queries and keys (0: that side is left out)
  int waves[2];       // of a workgroup's, those that take queries, then those that take keys
  int half;           // pairs of a head
  int lg;             // lanes of a row, as a power of 2
  int axes;
  int first[kMaxAxes + 1];  // first pair of each axis
  const void* pos;    // [tokens, axes], or [batch, tokens, axes] with pos_batch
  int pos_kind;       // 0 int32, 1 int64, 2 fp32
  int64_t pos_batch;
  const double* freq; // radians per position of each pair, or NULL: from theta
  double log2_theta;
  float sign;         // -1 turns back
  float eps;
  int weight_dtype;
  const void* w[2];   // NULL: ones
};

// 8 bytes in memory at the alignment of a 2- or 4-byte element.
template <int ALIGN>
struct Bytes8;
template <>
struct Bytes8<2> {
  typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2)));
};
template <>
struct Bytes8<4> {
  typedef uint32_t type __attribute__((ext_vector_type(2), aligned(4)));
};

// VP elements as they are in memory, at any alignment: 8 or 16 bytes.
template <class T, int VP>
struct Raw {
  static constexpr bool WIDE = VP * sizeof(T) == 16;
  static_assert(WIDE || VP * sizeof(T) == 8, "8 or 16 bytes");
  using raw = typename std::conditional<WIDE, typename Vec<T>::raw, typename Bytes8<sizeof(T)>::type>::type;
  static constexpr int WORDS = WIDE ? 4 : 2;
  // the first n, the rest 0
  static __device__ __forceinline__ raw load(const T* p, int n) {
    if (n >= VP) return *(const raw*)p;
    raw r;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) r[i] = 0;
#pragma unroll
    for (int i = 0; i < VP; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 4)
          r[i] = __float_as_uint(p[i]);
        else
          r[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (16 * (i & 1));
      }
    return r;
  }
  static __device__ __forceinline__ void unpack(const raw& r, float (&v)[VP]) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(r[i]);
      } else if constexpr (std::is_same<T, uint16_t>::value) {
        v[2 * i] = __uint_as_float(r[i] << 16);
        v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
      } else {
        const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)r[i]);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, int n, const float (&v)[VP]) {
    if (n >= VP) {
      raw r;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        if constexpr (sizeof(T) == 4)
          r[i] = __float_as_uint(v[i]);
        else if constexpr (std::is_same<T, uint16_t>::value)
          r[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
        else
          r[i] = pack2_f16(v[2 * i], v[2 * i + 1]);
      }
      *(raw*)p = r;
    } else {
#pragma unroll
      for (int i = 0; i < VP; ++i)
        if (i < n) put(p + i, v[i]);
    }
  }
};

// The n pairs of a lane that begin at pair p0 of a row, as they are in memory.
template <class T, int VP, bool IL>
struct Pairs {
  using R = Raw<T, VP>;
  typename R::raw lo, hi;
  __device__ __forceinline__ void load(const T* x, int p0, int n, int half) {
    lo = R::load(x + (IL ? 2 * p0 : p0), IL ? 2 * n : n);
    hi = R::load(x + (IL ? 2 * p0 + VP : half + p0), IL ? 2 * n - VP : n);
  }
  __device__ __forceinline__ void unpack(float (&a)[VP], float (&b)[VP]) const {
    if constexpr (IL) {
      float u[VP], v[VP];
      R::unpack(lo, u);
      R::unpack(hi, v);
#pragma unroll
      for (int i = 0; i < VP / 2; ++i) {
        a[i] = u[2 * i];
        b[i] = u[2 * i + 1];
        a[VP / 2 + i] = v[2 * i];
        b[VP / 2 + i] = v[2 * i + 1];
      }
    } else {
      R::unpack(lo, a);
      R::unpack(hi, b);
    }
  }
  static __device__ __forceinline__ void store(T* x, int p0, int n, int half, const float (&a)[VP], const float (&b)[VP]) {
    if constexpr (IL) {
      float u[VP], v[VP];
#pragma unroll
      for (int i = 0; i < VP / 2; ++i) {
        u[2 * i] = a[i];
        u[2 * i + 1] = b[i];
        v[2 * i] = a[VP / 2 + i];
        v[2 * i + 1] = b[VP / 2 + i];
      }
      R::store(x + 2 * p0, 2 * n, u);
      R::store(x + 2 * p0 + VP, 2 * n - VP, v);
    } else {
      R::store(x + p0, n, a);
      R::store(x + half + p0, n, b);
    }
  }
};

// Sum over the 2^lg lanes of a row.
__device__ __forceinline__ float row_sum(float v, int lg) {
  for (int m = 0; m < lg; ++m) v += __shfl_xor(v, 1 << m, 64);
  return v;
}

// Turns per position and the axis of a lane's pairs (lane and lane + 64).
struct Turns {
  double f[2];
  int axis[2];
  __device__ __forceinline__ void init(const RotaryShape& s, int lane) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int p = lane + 64 * q;
      int a = 0;
      for (int i = 1; i < s.axes; ++i) a = p >= s.first[i] ? i : a;
      axis[q] = a;
      f[q] = 0.0;
      if (p < s.half) {
        const int n = s.first[a + 1] - s.first[a];
        const double rad = s.freq ? s.freq[p] : exp2(-s.log2_theta * ((double)(p - s.first[a]) / (double)n));
        f[q] = rad * 0.15915494309189533577;  // 1 / 2 pi
      }
    }
  }
  // cos and sin of the token's pairs into LDS
  __device__ __forceinline__ void turn(const RotaryShape& s, int64_t at, int lane, float* cs, float* sn) const {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int p = lane + 64 * q;
      if (p < s.half) {
        const int64_t i = at + axis[q];
        const double x = s.pos_kind == 0   ? (double)((const int32_t*)s.pos)[i]
                         : s.pos_kind == 1 ? (double)((const int64_t*)s.pos)[i]
                                           : (double)((const float*)s.pos)[i];
        // the nearest quarter turn and what is left, at most an eighth: rounded to 32
        // bits it keeps its relative error, and with it a sine or cosine near 0
        const double t = x * f[q], quarter = rint(4.0 * t);
        float c, n;
        sincospif(2.f * (float)(t - 0.25 * quarter), &n, &c);
        const double k = quarter - 4.0 * floor(0.25 * quarter);  // 0 .. 3
        const bool odd = k == 1.0 || k == 3.0;
        const float cq = odd ? n : c, nq = odd ? c : n;
        cs[p] = k == 1.0 || k == 2.0 ? -cq : cq;
        sn[p] = k >= 2.0 ? -s.sign * nq : s.sign * nq;
      }
    }
  }
};

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (w == nullptr) return 1.f;
  return dtype == 0 ? ((const float*)w)[i] : dtype == 1 ? bf16_to_f32(((const uint16_t*)w)[i]) : (float)((const _Float16*)w)[i];
}
// A lane's weights of queries (side 0) or keys.
template <int VP, bool IL>
__device__ __forceinline__ void load_weights(const RotaryShape& s, int side, int p0, float (&a)[VP], float (&b)[VP]) {
#pragma unroll
  for (int i = 0; i < VP; ++i) {
    const int p = p0 + i;
    a[i] = p < s.half ? weight_at(s.w[side], s.weight_dtype, IL ? 2 * p : p) : 0.f;
    b[i] = p < s.half ? weight_at(s.w[side], s.weight_dtype, IL ? 2 * p + 1 : p + s.half) : 0.f;
  }
}

// A wave's way over its side: the passes over a token's heads, 64 / 2^lg rows each, of the tokens
// first, first + step, ...
struct Walk {
  int side, heads, groups, group, passes;
  int64_t step, rows;
  int64_t row;     // token, and where it lies
  int64_t b, t;
  int pass;
  int tokens;
  __device__ __forceinline__ Walk(const RotaryShape& s, int wave, int lane) {
    side = wave >= s.waves[0];
    heads = s.heads[side];
    group = lane >> s.lg;
    groups = 64 >> s.lg;
    passes = (heads + groups - 1) / groups;
    rows = s.rows;
    tokens = s.tokens;
    step = (int64_t)gridDim.x * s.waves[side];
    pass = 0;
    place((int64_t)blockIdx.x * s.waves[side] + (side ? wave - s.waves[0] : wave));
  }
  __device__ __forceinline__ void place(int64_t r) {
    row = r;
    b = r / tokens;
    t = r - b * tokens;
  }
  __device__ __forceinline__ bool done() const { return row >= rows; }
  __device__ __forceinline__ void next() {
    if (++pass == passes) {
      pass = 0;
      place(row + step);
    }
  }
  __device__ __forceinline__ int head() const { return pass * groups + group; }
  // this lane's row, and its pairs there (0: no row)
  template <class T>
  __device__ __forceinline__ const T* at(const HeadsView& v) const {
    return (const T*)v.p + b * v.batch + t * v.token + (int64_t)head() * v.head;
  }
  __device__ __forceinline__ int pairs(int n) const { return !done() && head() < heads ? n : 0; }
};
// cos and sin of this lane's pairs of the walk's token
template <int VP>
__device__ __forceinline__ void angles(const Turns& turns, const RotaryShape& s, const Walk& w, int lane, float* cs,
                                       float* sn, int p0, int n, float (&c)[VP], float (&z)[VP]) {
  turns.turn(s, w.b * s.pos_batch + w.t * s.axes, lane, cs, sn);
  wave_sync();
#pragma unroll
  for (int i = 0; i < VP; ++i) {
    const bool in = i < n;
    c[i] = in ? cs[p0 + i] : 0.f;
    z[i] = in ? sn[p0 + i] : 0.f;
  }
  wave_sync();
}

template <class T, int VP, bool IL, bool NORM>
__global__ __launch_bounds__(64 * kRotaryWaves) void k_rotary(RotaryShape s, HeadsView q, HeadsView k, T* yq, T* yk) {
  using P = Pairs<T, VP, IL>;
  __shared__ alignas(16) float s_cos[kRotaryWaves][kMaxHalf + VP], s_sin[kRotaryWaves][kMaxHalf + VP];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float *cs = s_cos[wave], *sn = s_sin[wave];
  const int p0 = (lane & ((1 << s.lg) - 1)) * VP, n = s.half - p0, d = 2 * s.half;  // this lane's pairs
  Walk w(s, wave, lane);
  const HeadsView v = w.side ? k : q;
  T* const y = w.side ? yk : yq;
  if (w.done() || w.heads == 0) return;
  P x;
  x.load(w.at<T>(v), p0, w.pairs(n), s.half);
  Turns turns;
  turns.init(s, lane);
  float wa[VP], wb[VP], c[VP], z[VP];
  if constexpr (NORM) load_weights<VP, IL>(s, w.side, p0, wa, wb);
  while (!w.done()) {
    if (w.pass == 0) angles<VP>(turns, s, w, lane, cs, sn, p0, n, c, z);
    float a[VP], b[VP], ya[VP], yb[VP];
    x.unpack(a, b);
    const int h = w.head();
    T* const to = h < w.heads ? y + (w.row * w.heads + h) * d : nullptr;
    w.next();
    x.load(w.at<T>(v), p0, w.pairs(n), s.half);
    if constexpr (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VP; ++i) sum += a[i] * a[i] + b[i] * b[i];
      const float r = rsqrtf(row_sum(sum, s.lg) / (float)d + s.eps);
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        a[i] *= r * wa[i];
        b[i] *= r * wb[i];
      }
    }
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      ya[i] = a[i] * c[i] - b[i] * z[i];
      yb[i] = b[i] * c[i] + a[i] * z[i];
    }
    if (to) P::store(to, p0, n, s.half, ya, yb);
  }
}

// The gradient through turn and norm.  dwq, dwk: sums of a workgroup,
// parts[workgroup][2][d] (NULL: none asked for); dxq or dxk NULL: not written.
template <class T, int VP, bool IL>
__global__ __launch_bounds__(64 * kRotaryWaves) void k_rotary_norm_grad(RotaryShape s, HeadsView q, HeadsView k,
                                                                        HeadsView gq, HeadsView gk, T* dxq, T* dxk,
                                                                        float* parts) {
  using P = Pairs<T, VP, IL>;
  __shared__ alignas(16) float s_cos[kRotaryWaves][kMaxHalf + VP], s_sin[kRotaryWaves][kMaxHalf + VP];
  __shared__ float s_dw[kRotaryWaves][2 * kMaxHalf];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float *cs = s_cos[wave], *sn = s_sin[wave];
  const int p0 = (lane & ((1 << s.lg) - 1)) * VP, n = s.half - p0, d = 2 * s.half;
  Walk w(s, wave, lane);
  const HeadsView v = w.side ? k : q, g = w.side ? gk : gq;
  T* const dx = w.side ? dxk : dxq;
  float da[VP], db[VP];
#pragma unroll
  for (int i = 0; i < VP; ++i) da[i] = db[i] = 0.f;
  if (!w.done() && w.heads > 0) {
    P x, y;
    x.load(w.at<T>(v), p0, w.pairs(n), s.half);
    y.load(w.at<T>(g), p0, w.pairs(n), s.half);
    Turns turns;
    turns.init(s, lane);
    float wa[VP], wb[VP], c[VP], z[VP];
    load_weights<VP, IL>(s, w.side, p0, wa, wb);
    while (!w.done()) {
      if (w.pass == 0) angles<VP>(turns, s, w, lane, cs, sn, p0, n, c, z);
      float xa[VP], xb[VP], ga[VP], gb[VP];
      x.unpack(xa, xb);
      y.unpack(ga, gb);
      const int h = w.head();
      T* const to = dx != nullptr && h < w.heads ? dx + (w.row * w.heads + h) * d : nullptr;
      w.next();
      x.load(w.at<T>(v), p0, w.pairs(n), s.half);
      y.load(w.at<T>(g), p0, w.pairs(n), s.half);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VP; ++i) sum += xa[i] * xa[i] + xb[i] * xb[i];
      // (rows that are none are 0, and have no part in dw)
      const float r = h < w.heads ? rsqrtf(row_sum(sum, s.lg) / (float)d + s.eps) : 0.f;
      // dx = r g w - x r^3 mean(g w x)
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        const float ta = ga[i] * c[i] + gb[i] * z[i], tb = gb[i] * c[i] - ga[i] * z[i];
        const float ua = ta * xa[i], ub = tb * xb[i];
        da[i] = fmaf(ua, r, da[i]);
        db[i] = fmaf(ub, r, db[i]);
        dot = fmaf(ua, wa[i], dot);
        dot = fmaf(ub, wb[i], dot);
        ga[i] = ta * (wa[i] * r);
        gb[i] = tb * (wb[i] * r);
      }
      const float less = -(row_sum(dot, s.lg) / (float)d) * r * r * r;
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        ga[i] = fmaf(xa[i], less, ga[i]);
        gb[i] = fmaf(xb[i], less, gb[i]);
      }
      if (to) P::store(to, p0, n, s.half, ga, gb);
    }
  }
  if (parts == nullptr) return;
  // over the groups of the wave, then over the side's waves, in this order
  for (int m = 1 << s.lg; m < 64; m <<= 1)
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      da[i] += __shfl_xor(da[i], m, 64);
      db[i] += __shfl_xor(db[i], m, 64);
    }
  if (w.group == 0) {
#pragma unroll
    for (int i = 0; i < VP; ++i)
      if (i < n) {
        const int p = p0 + i;
        s_dw[wave][IL ? 2 * p : p] = da[i];
        s_dw[wave][IL ? 2 * p + 1 : p + s.half] = db[i];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * d; i += 64 * kRotaryWaves) {
    const int side = i >= d, from = side ? s.waves[0] : 0;
    float sum = 0.f;
    for (int u = 0; u < s.waves[side]; ++u) sum += s_dw[from + u][i - side * d];
    parts[(int64_t)blockIdx.x * 2 * d + i] = sum;
  }
}

// dw = sum of the workgroups' parts: 64 columns a workgroup, its 16 waves take
// every 16th part each.
constexpr int kDwWaves = 16;
template <class W>
__global__ __launch_bounds__(64 * kDwWaves) void k_rotary_dw(const float* parts, int n, int d, W* dwq, W* dwk) {
  __shared__ float s_sum[kDwWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  float v = 0.f;
  if (col < 2 * d)
#pragma unroll 8
    for (int i = wave; i < n; i += kDwWaves) v += parts[(int64_t)i * 2 * d + col];
  s_sum[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && col < 2 * d) {
    v = 0.f;
    for (int w = 0; w < kDwWaves; ++w) v += s_sum[w][lane];
    W* out = col < d ? dwq : dwk;
    if (out) put(out + (col < d ? col : col - d), v);
  }
}

}  // namespace mec
