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
// written), all else is registers.  A wave takes a token with all of its query
// and key heads, so that the angles of a token are formed once, one pair a
// lane, and handed to the lanes that need them through LDS.  In a head's row a
// lane holds VP pairs, both halves of each, so that the turn crosses no lanes;
// a group of 2^lg lanes is a row, and only the norm's sum of squares crosses
// them.  ROWS rows of a group are in flight at once.
#pragma once
#include "mec_vec.h"

namespace mec {

constexpr int kRotaryWaves = 4;
constexpr int kMaxAxes = 8;
constexpr int kMaxHalf = 128;  // pairs of a head

// Heads as the callers give them: element (b, t, h, i) at p[b * batch + t * token + h * head + i].
struct HeadsView {
  const void* p;
  int64_t batch, token, head;
};

struct RotaryShape {
  int64_t rows;       // batch * tokens
  int tokens;
  int heads[2];       // of queries and keys (0: that side is left out)
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

// VP elements at any alignment, the first n of them (the rest 0).
template <class T, int VP>
__device__ __forceinline__ void load_some(const T* p, int n, float (&v)[VP]) {
  if constexpr (VP * sizeof(T) == 16) {
    load_row(p, n, v);
  } else {
    using raw = typename Bytes8<sizeof(T)>::type;
    static_assert(VP * sizeof(T) == 8, "8 or 16 bytes");
    if (n >= VP) {
      const raw r = *(const raw*)p;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
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
    } else {
#pragma unroll
      for (int i = 0; i < VP; ++i) v[i] = i < n ? value(p[i]) : 0.f;
    }
  }
}
template <class T, int VP>
__device__ __forceinline__ void store_some(T* p, int n, const float (&v)[VP]) {
  if constexpr (VP * sizeof(T) == 16) {
    store_row(p, n, v);
  } else {
    using raw = typename Bytes8<sizeof(T)>::type;
    if (n >= VP) {
      raw r;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
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
}

// The n pairs of a lane that begin at pair p0 of the row x.
template <class T, int VP, bool IL>
__device__ __forceinline__ void load_pairs(const T* x, int p0, int n, int half, float (&a)[VP], float (&b)[VP]) {
  if constexpr (IL) {
    float u[VP], v[VP];
    load_some<T, VP>(x + 2 * p0, 2 * n, u);
    load_some<T, VP>(x + 2 * p0 + VP, 2 * n - VP, v);
#pragma unroll
    for (int i = 0; i < VP / 2; ++i) {
      a[i] = u[2 * i];
      b[i] = u[2 * i + 1];
      a[VP / 2 + i] = v[2 * i];
      b[VP / 2 + i] = v[2 * i + 1];
    }
  } else {
    load_some<T, VP>(x + p0, n, a);
    load_some<T, VP>(x + half + p0, n, b);
  }
}
template <class T, int VP, bool IL>
__device__ __forceinline__ void store_pairs(T* x, int p0, int n, int half, const float (&a)[VP], const float (&b)[VP]) {
  if constexpr (IL) {
    float u[VP], v[VP];
#pragma unroll
    for (int i = 0; i < VP / 2; ++i) {
      u[2 * i] = a[i];
      u[2 * i + 1] = b[i];
      v[2 * i] = a[VP / 2 + i];
      v[2 * i + 1] = b[VP / 2 + i];
    }
    store_some<T, VP>(x + 2 * p0, 2 * n, u);
    store_some<T, VP>(x + 2 * p0 + VP, 2 * n - VP, v);
  } else {
    store_some<T, VP>(x + p0, n, a);
    store_some<T, VP>(x + half + p0, n, b);
  }
}

// Sum over the 2^lg lanes of a row.
__device__ __forceinline__ float row_sum(float v, int lg) {
  for (int m = 0; m < lg; ++m) v += __shfl_xor(v, 1 << m, 64);
  return v;
}

// What the lanes of a wave wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
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

// A wave's way over the tokens: `first`, `first + step`, ...
struct TokenWalk {
  int64_t first, step;
  __device__ __forceinline__ TokenWalk() {
    first = (int64_t)blockIdx.x * kRotaryWaves + (threadIdx.x >> 6);
    step = (int64_t)gridDim.x * kRotaryWaves;
  }
};

template <class T, int VP, bool IL, bool NORM>
__global__ __launch_bounds__(64 * kRotaryWaves) void k_rotary(RotaryShape s, HeadsView q, HeadsView k, T* yq, T* yk) {
  constexpr int ROWS = 2;
  __shared__ alignas(16) float s_cos[kRotaryWaves][kMaxHalf + VP], s_sin[kRotaryWaves][kMaxHalf + VP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float *cs = s_cos[wave], *sn = s_sin[wave];
  const int p0 = (lane & ((1 << s.lg) - 1)) * VP, n = s.half - p0;  // this lane's pairs
  const int group = lane >> s.lg, groups = 64 >> s.lg;
  const int heads = s.heads[0] + s.heads[1], d = 2 * s.half;
  Turns turns;
  turns.init(s, lane);
  float wa[2][VP], wb[2][VP];
  if constexpr (NORM) {
    load_weights<VP, IL>(s, 0, p0, wa[0], wb[0]);
    load_weights<VP, IL>(s, 1, p0, wa[1], wb[1]);
  }
  const TokenWalk walk;
  for (int64_t row = walk.first; row < s.rows; row += walk.step) {
    const int64_t b = row / s.tokens, t = row - b * s.tokens;
    turns.turn(s, b * s.pos_batch + t * s.axes, lane, cs, sn);
    wave_sync();
    float c[VP], z[VP];
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const bool in = i < n;
      c[i] = in ? cs[p0 + i] : 0.f;
      z[i] = in ? sn[p0 + i] : 0.f;
    }
    wave_sync();
    for (int h0 = group; h0 < heads; h0 += ROWS * groups) {
      float xa[ROWS][VP], xb[ROWS][VP];
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int h = h0 + u * groups;
        const bool key = h >= s.heads[0];
        const HeadsView& v = key ? k : q;
        const T* x = (const T*)v.p + b * v.batch + t * v.token + (int64_t)(key ? h - s.heads[0] : h) * v.head;
        load_pairs<T, VP, IL>(x, p0, h < heads ? n : 0, s.half, xa[u], xb[u]);
      }
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int h = h0 + u * groups;
        const bool key = h >= s.heads[0];
        if constexpr (NORM) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < VP; ++i) sum += xa[u][i] * xa[u][i] + xb[u][i] * xb[u][i];
          const float r = rsqrtf(row_sum(sum, s.lg) / (float)d + s.eps);
#pragma unroll
          for (int i = 0; i < VP; ++i) {
            xa[u][i] *= r * (key ? wa[1][i] : wa[0][i]);
            xb[u][i] *= r * (key ? wb[1][i] : wb[0][i]);
          }
        }
        float ya[VP], yb[VP];
#pragma unroll
        for (int i = 0; i < VP; ++i) {
          ya[i] = xa[u][i] * c[i] - xb[u][i] * z[i];
          yb[i] = xb[u][i] * c[i] + xa[u][i] * z[i];
        }
        if (h < heads) {
          T* y = key ? yk + (row * s.heads[1] + (h - s.heads[0])) * d : yq + (row * s.heads[0] + h) * d;
          store_pairs<T, VP, IL>(y, p0, n, s.half, ya, yb);
        }
      }
    }
  }
}

// The gradient through turn and norm.  dwq, dwk: sums of a workgroup,
// parts[workgroup][2][d] (NULL: none asked for); dxq or dxk NULL: not written.
template <class T, int VP, bool IL>
__global__ __launch_bounds__(64 * kRotaryWaves) void k_rotary_norm_grad(RotaryShape s, HeadsView q, HeadsView k,
                                                                        HeadsView gq, HeadsView gk, T* dxq, T* dxk,
                                                                        float* parts) {
  __shared__ alignas(16) float s_cos[kRotaryWaves][kMaxHalf + VP], s_sin[kRotaryWaves][kMaxHalf + VP];
  __shared__ float s_dw[kRotaryWaves][2 * kMaxHalf];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float *cs = s_cos[wave], *sn = s_sin[wave];
  const int p0 = (lane & ((1 << s.lg) - 1)) * VP, n = s.half - p0;
  const int group = lane >> s.lg, groups = 64 >> s.lg;
  const int heads = s.heads[0] + s.heads[1], d = 2 * s.half;
  Turns turns;
  turns.init(s, lane);
  float wa[2][VP], wb[2][VP], da[2][VP], db[2][VP];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    load_weights<VP, IL>(s, e, p0, wa[e], wb[e]);
#pragma unroll
    for (int i = 0; i < VP; ++i) da[e][i] = db[e][i] = 0.f;
  }
  const TokenWalk walk;
  for (int64_t row = walk.first; row < s.rows; row += walk.step) {
    const int64_t b = row / s.tokens, t = row - b * s.tokens;
    turns.turn(s, b * s.pos_batch + t * s.axes, lane, cs, sn);
    wave_sync();
    float c[VP], z[VP];
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const bool in = i < n;
      c[i] = in ? cs[p0 + i] : 0.f;
      z[i] = in ? sn[p0 + i] : 0.f;
    }
    wave_sync();
    for (int h = group; h < heads; h += groups) {
      const bool key = h >= s.heads[0];
      const int hh = key ? h - s.heads[0] : h;
      const HeadsView &v = key ? k : q, &g = key ? gk : gq;
      float xa[VP], xb[VP], ga[VP], gb[VP];
      load_pairs<T, VP, IL>((const T*)v.p + b * v.batch + t * v.token + (int64_t)hh * v.head, p0, n, s.half, xa, xb);
      load_pairs<T, VP, IL>((const T*)g.p + b * g.batch + t * g.token + (int64_t)hh * g.head, p0, n, s.half, ga, gb);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VP; ++i) sum += xa[i] * xa[i] + xb[i] * xb[i];
      const float r = rsqrtf(row_sum(sum, s.lg) / (float)d + s.eps);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        const float ta = ga[i] * c[i] + gb[i] * z[i], tb = gb[i] * c[i] - ga[i] * z[i];
        xa[i] *= r;
        xb[i] *= r;
        const float wqa = ta * xa[i], wqb = tb * xb[i];
        da[0][i] += key ? 0.f : wqa;
        db[0][i] += key ? 0.f : wqb;
        da[1][i] += key ? wqa : 0.f;
        db[1][i] += key ? wqb : 0.f;
        ga[i] = ta * (key ? wa[1][i] : wa[0][i]);
        gb[i] = tb * (key ? wb[1][i] : wb[0][i]);
        dot += ga[i] * xa[i] + gb[i] * xb[i];
      }
      const float mean = row_sum(dot, s.lg) / (float)d;
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        ga[i] = r * (ga[i] - xa[i] * mean);
        gb[i] = r * (gb[i] - xb[i] * mean);
      }
      T* dx = key ? dxk : dxq;
      if (dx) store_pairs<T, VP, IL>(dx + (row * s.heads[key] + hh) * d, p0, n, s.half, ga, gb);
    }
  }
  if (parts == nullptr) return;
  // over the groups of the wave, then over the waves, in this order
  for (int m = 1 << s.lg; m < 64; m <<= 1)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        da[e][i] += __shfl_xor(da[e][i], m, 64);
        db[e][i] += __shfl_xor(db[e][i], m, 64);
      }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (group == 0) {
#pragma unroll
      for (int i = 0; i < VP; ++i)
        if (i < n) {
          const int p = p0 + i;
          s_dw[wave][IL ? 2 * p : p] = da[e][i];
          s_dw[wave][IL ? 2 * p + 1 : p + s.half] = db[e][i];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < d; i += 64 * kRotaryWaves) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kRotaryWaves; ++w) v += s_dw[w][i];
      parts[((int64_t)blockIdx.x * 2 + e) * d + i] = v;
    }
    __syncthreads();
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
