// Attention of short sequences, whose tiles fit into LDS as a whole: the texts and
// patches of a contrastive batch.  A workgroup takes all tokens of one key head.
//
// Beside the kernels that walk over tiles this saves their barriers, their second
// reading of the inputs in the backward, and the time until a tile has arrived,
// which here is spent once: everything is on its way to LDS before the first
// product, by loads that pass no registers.
#pragma once
#include <climits>

#include "mec_attn_strict.h"

namespace mec {
namespace attn {

// most waves of a workgroup: registers for 3 or 2 on a SIMD
constexpr int whole_waves(int steps, int size) { return steps <= 4 && size == 2 ? 12 : 8; }
constexpr int whole_steps(int size) { return size == 2 ? 6 : 4; }  // of 16 features: the widest heads
constexpr int kWholeLds = 160 * 1024;  // of a CU

extern __shared__ __align__(16) char s_whole[];

// Rows [0, valid) of a head into `rows` rows (a multiple of 32), the rest as zeros: in
// blocks of 32, with as much room after each for the block of another matrix, which is
// then at a distance that the reading instructions hold.
template <class T, int DB>
__device__ __forceinline__ void fetch(Lds* tile, const View& v, int64_t b, int h, int valid, int rows, int d, int wave,
                                      int waves) {
  using Tl = Tile<T, DB>;
  constexpr int VPR = Tl::VPR;
  const char* base = (const char*)((const T*)v.p + b * v.batch + (int64_t)h * v.head);
  const int64_t pitch = v.token * (int64_t)sizeof(T);
  const int lane = threadIdx.x & 63, blocks = rows * VPR / 64;
  if (d % Tl::EPV == 0 && ((uintptr_t)base & 15) == 0 && (pitch & 15) == 0 && pitch < (1 << 20)) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
    for (int i = wave; i < blocks; i += waves) {
      // lane l fills place l of the i-th 64, VPR / 2 of which are a block
      const int at = i * 64 + lane, row = at / VPR, vec = (at % VPR) ^ Tl::swz(row);
      const uint32_t off = row < valid && vec * Tl::EPV < d ? (uint32_t)(row * (int)pitch + vec * 16) : OOB;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(tile + (i + i / (VPR / 2) * (VPR / 2)) * 1024),
                                               16, off, 0, 0, 0);
    }
  } else {
    for (int i = wave; i < blocks; i += waves) {
      const int at = i * 64 + lane, row = at / VPR, vec = (at % VPR) ^ Tl::swz(row);
      const u32x4 r = load_raw((const T*)(base + row * pitch) + vec * Tl::EPV, row < valid ? d - vec * Tl::EPV : 0);
      *(__attribute__((address_space(3))) u32x4*)(tile + (at + i / (VPR / 2) * 32 * VPR) * 16) = r;
    }
  }
}

// The forward: each wave has a block of 32 rows (r = query * group + head), as in
// k_attn_forward; LDS holds K and V.
template <class T, int KS>
__global__ __launch_bounds__(64 * whole_waves(KS, sizeof(T)), sizeof(T) == 4 || KS > 6 ? 2 : KS > 4 ? 3 : 5) void
k_attn_whole_forward(Problem a, Items items, T* out, float* lse) {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  constexpr int DB = (KS + 1) / 2;
  using Tl = Tile<T, DB>;
  constexpr int BLOCK = 32 * Tl::RB;
  int64_t id;
  int tile;
  if (!items.take(a.pairs, 1, id, tile)) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  typename Tl::At lane_at(lane);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int64_t b = id / a.key_heads;
  const int kh = (int)(id - b * a.key_heads);
  const int nq = a.nq(b), nk = a.nk(b), shift = nk - nq;
  Lds* const tk = (Lds*)s_whole;
  const int first = 32 * wave, row = first + (lane & 31), rows = a.queries * a.group;
  const int qi = row / a.group, qh = kh * a.group + row % a.group;
  const bool live = qi < nq;
  const int see = a.causal ? min(nk, qi + shift + 1) : nk;
  const int all = a.causal ? min(nk, first / a.group + shift + 1) : nk;
  const int end = first / a.group >= nq ? 0 : a.causal ? min(nk, min((first + 31) / a.group, nq - 1) + shift + 1) : nk;
  Frag q[KS];
  if (nq > 0 && nk > 0) {
    const int nk32 = (nk + 31) & ~31;
    fetch<T, DB>(tk, a.k, b, kh, nk, nk32, a.d, wave, waves);
    fetch<T, DB>(tk + BLOCK, a.v, b, kh, nk, nk32, a.d, wave, waves);
    const T* p = (const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)qh * a.q.head;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = O::load_row(p, live, s, half, a.d);
  }
  loads_done();
  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();
  float m = -kInf, l = 0.f;
  Lds* at = tk;
  for (int key0 = 0; key0 < end; key0 += 32, at += 2 * BLOCK) {
    lane_at.again();
    f32x16 s = zero16();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = O::mma(Tl::row(at, 0, ks, lane_at), q[ks], s);
    if (key0 + 32 > all) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = key0 + 8 * (e >> 2) + 4 * half + (e & 3) < see ? s[e] : -kInf;
    }
    grow<O>(s, a.c, m, l, o);
    const float ref = (m == -kInf ? 0.f : m) - O::BIAS;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = fast_exp2(fmaf(s[e], a.c, -ref));
      l += s[e];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const Frag p = O::pack(s, x);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = O::mma(Tl::col(at + BLOCK, 16 * x, db, lane_at), p, o[db]);
    }
  }
  if (a.causal && any_nan<O>(o)) {
    float again[16 * DB + 2];
    strict_forward<T, KS>((const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)qh * a.q.head, live,
                          (const T*)a.k.p + b * a.k.batch + (int64_t)kh * a.k.head, a.k.token,
                          (const T*)a.v.p + b * a.v.batch + (int64_t)kh * a.v.head, a.v.token, a.d,
                          Range{0, (end + 31) / 32, 1, 32}, end, see, a.c, again);
    take<DB>(o, again);
    m = again[16 * DB];
    l = again[16 * DB + 1];
  }
  l += other_half(l);
  if (!live || l == 0.f) {
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = zero16();
  }
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  if (lse && half == 0 && row < rows)
    lse[(b * a.heads + qh) * (int64_t)a.queries + qi] = l == 0.f ? kInf : m - O::BIAS + log2f(l);
  __syncthreads();  // (keys and values are no longer read)
  store_rows<T, DB>(tk + wave * BLOCK, o, inv, a.d, lane, [&](int r) -> T* {
    const int to = first + r;
    return to < rows ? out + ((b * a.queries + to / a.group) * a.heads + kh * a.group + to % a.group) * (int64_t)a.d
                     : nullptr;
  });
}

// The gradients of one head (heads == key_heads).  Each wave has a block of 32 queries
// and one of 32 keys: first S^T, dP^T and dQ^T of the queries as in k_attn_dq, with
// delta made whole (see there), then S, dP, dV^T and dK^T of the keys as in k_attn_dkv.
// LDS: K, V, Q, dO, and lse and delta of the queries.
template <class T, int KS>
__global__ __launch_bounds__(64 * whole_waves(KS, sizeof(T))) void k_attn_whole_grad(Problem a, Items items, const T* out,
                                                                                     const float* lse,
                                                                                     T* dq, T* dk, T* dv) {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  constexpr int DB = (KS + 1) / 2;
  using Tl = Tile<T, DB>;
  // a wave's keys and values, in registers; of fp32 and of wide heads they are read from LDS
  constexpr bool HELD = !O::F32 && DB <= 2;
  // see Backward: d + eps is delta, and dq is corrected by the sum of the rounded ds times the mean key
  constexpr bool MEAN = !O::F32 && DB <= 2, TWICE = !O::F32 && DB > 2;
  int64_t id;
  int tile;
  if (!items.take(a.pairs, 1, id, tile)) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  typename Tl::At lane_at(lane);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int64_t b = id / a.key_heads;
  const int h = (int)(id - b * a.key_heads);
  const int nq = a.nq(b), nk = a.nk(b), shift = nk - nq;
  const int q_rows = (a.queries + 31) & ~31, k_rows = (a.keys + 31) & ~31;
  // (blocks of K and V, and of Q and dO, in turn)
  constexpr int BLOCK = 32 * Tl::RB;
  Lds* const tk = (Lds*)s_whole;
  Lds* const tq = tk + 2 * k_rows * Tl::RB;
  typedef __attribute__((address_space(3))) float LdsFloat;
  typedef __attribute__((address_space(3))) f32x4 LdsFour;
  LdsFloat* const s_lse = (LdsFloat*)(tq + 2 * q_rows * Tl::RB);
  LdsFloat* const s_delta = s_lse + q_rows;
  Lds* const my_k = tk + 2 * wave * BLOCK;
  Lds* const my_q = tq + 2 * wave * BLOCK;
  const int64_t head0 = (b * a.heads + h) * (int64_t)a.queries;  // of lse
  const int first = 32 * wave;                                  // of the wave's queries, and of its keys
  const int qi = first + (lane & 31), key = qi;
  const bool live = qi < nq;
  const int end = first >= nq || nk == 0 ? 0 : a.causal ? min(nk, min(first + 31, nq - 1) + shift + 1) : nk;
  Frag o[O::F32 || TWICE ? 1 : KS];  // (the result: on its way from memory along with the tiles)
  float l2 = kInf;
  if (nq > 0 && nk > 0) {
    // (blocks that the lengths leave empty are not touched)
    const int nq32 = (nq + 31) & ~31, nk32 = (nk + 31) & ~31;
    fetch<T, DB>(tk, a.k, b, h, nk, nk32, a.d, wave, waves);
    fetch<T, DB>(tq, a.q, b, h, nq, nq32, a.d, wave, waves);
    fetch<T, DB>(tk + BLOCK, a.v, b, h, nk, nk32, a.d, wave, waves);
    fetch<T, DB>(tq + BLOCK, a.g, b, h, nq, nq32, a.d, wave, waves);
    if (live) l2 = lse[head0 + qi];
    if constexpr (MEAN) {
      const T* po = out + ((b * a.queries + qi) * a.heads + h) * (int64_t)a.d;
#pragma unroll
      for (int s = 0; s < KS; ++s) o[s] = O::load_row(po, live, s, half, a.d);
    }
    if (half == 0 && first < nq) s_lse[qi] = l2 - O::GRAD_BIAS;
  }
  loads_done();
  Rows<T, DB> packed;  // dq
  {
    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = zero16();
    float dot = 0.f;
    if (end > 0) {
      const int see = a.causal ? min(nk, qi + shift + 1) : nk, all = a.causal ? min(nk, first + shift + 1) : nk;
      Frag q[KS], g[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        q[s] = Tl::row(my_q, 0, s, lane_at);
        g[s] = Tl::row(my_q + BLOCK, 0, s, lane_at);
        if constexpr (MEAN) dot += O::dot(g[s], o[s]);
        if constexpr (O::F32)
          dot += O::dot(g[s], O::load_row(out + ((b * a.queries + qi) * a.heads + h) * (int64_t)a.d, live, s, half, a.d));
      }
      dot += other_half(dot);
      f32x16 mean[MEAN ? DB : 1];
#pragma unroll
      for (int db = 0; db < (MEAN ? DB : 1); ++db) mean[db] = zero16();
      float eps = 0.f, eps16 = 0.f;
      GradUnit<O> unit;  // of them and of acc
      for (int walk = TWICE ? 0 : 1; walk < 2; ++walk) {
        Lds* at = tk;
        for (int key0 = 0; key0 < end; key0 += 32, at += 2 * BLOCK) {
          lane_at.again();
          f32x16 s = zero16(), p = zero16();
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            s = O::mma(Tl::row(at, 0, ks, lane_at), q[ks], s);
            p = O::mma(Tl::row(at + BLOCK, 0, ks, lane_at), g[ks], p);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[e] = fast_exp2(fmaf(s[e], a.c, -l2));
            p[e] = s[e] * unit.times(p[e], dot);
          }
          if (key0 + 32 > all) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const bool in = key0 + 8 * (e >> 2) + 4 * half + (e & 3) < see;
              s[e] = in ? s[e] : 0.f;
              p[e] = in ? p[e] : 0.f;
            }
          }
          unit.fit(p, [&](float f) {
            scale_all(acc, f);
            eps *= f;
            eps16 *= f;
          });
          if (!O::F32) {
#pragma unroll
            for (int e = 0; e < 16; ++e) eps += p[e];
          }
          if (TWICE && walk == 0) continue;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const Frag ds = O::pack(p, x), ps = O::pack(s, x);
            if constexpr (MEAN) eps16 = O::add(ds, eps16);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const Frag kt = Tl::col(at, 16 * x, db, lane_at);
              acc[db] = O::mma(kt, ds, acc[db]);
              if constexpr (MEAN) mean[db] = O::mma(kt, ps, mean[db]);
            }
          }
        }
        if (TWICE && walk == 0) {
          if constexpr (O::F16) eps *= unit.back();
          dot += eps + other_half(eps);
          eps = 0.f;
        }
      }
      if constexpr (O::F16) {
        scale_all(acc, unit.back());
        eps *= unit.back();
        eps16 *= unit.back();
      }
      if constexpr (MEAN) {
        eps += other_half(eps);
        eps16 += other_half(eps16);
        dot += eps;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[db][e] -= eps16 * mean[db][e];
      }
      if (a.causal && any_nan<O>(acc)) {
        float again[16 * DB];
        strict_dq<T, KS>((const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)h * a.q.head,
                         (const T*)a.g.p + b * a.g.batch + (int64_t)qi * a.g.token + (int64_t)h * a.g.head, live,
                         (const T*)a.k.p + b * a.k.batch + (int64_t)h * a.k.head, a.k.token,
                         (const T*)a.v.p + b * a.v.batch + (int64_t)h * a.v.head, a.v.token, a.d,
                         Range{0, (end + 31) / 32, 1, 32}, end, see, a.c, l2, dot, again);
        take<DB>(acc, again);
      }
      if (!live || l2 == kInf)
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = zero16();
    }
    // (rows beyond the queries have none: 0 times a key or value that holds an inf is NaN)
    if (half == 0 && first < nq) s_delta[qi] = live ? dot : 0.f;
    packed.pack(acc, a.scale);
  }
  const auto to = [&](T* p, int n, int heads) {
    return [=](int r) -> T* { return first + r < n ? p + ((b * n + first + r) * heads + h) * (int64_t)a.d : nullptr; };
  };
  __syncthreads();  // delta is there, and other waves' keys and values are no longer read
  Frag k[HELD ? KS : 1], v[HELD ? KS : 1];
  if constexpr (HELD) {
    if (first < nk) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        k[s] = Tl::row(my_k, 0, s, lane_at);
        v[s] = Tl::row(my_k + BLOCK, 0, s, lane_at);
      }
    }
    if (dq) {
      __syncthreads();  // nor is any key or value
      if (first < a.queries) {
        packed.put(tk + wave * BLOCK, lane);
        Rows<T, DB>::flush(tk + wave * BLOCK, a.d, lane, to(dq, a.queries, a.heads));
      }
      __syncthreads();
    }
  }
  if (dk) {
    f32x16 ak[DB], av[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) ak[db] = av[db] = zero16();
    GradUnit<O> unit(O::GRAD_UNIT);  // of ak, beside that of the probabilities
    const int begin = first >= nk ? nq : a.causal ? max(0, first - shift) & ~31 : 0;
    const int all = a.causal ? first + 31 - shift : 0, seen = a.causal ? key - shift : 0;
    Lds* at = tq + begin * 2 * Tl::RB;
    for (int q0 = begin; q0 < nq; q0 += 32, at += 2 * BLOCK) {
      lane_at.again();
      f32x16 s = zero16(), p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 dl = *(LdsFour*)(s_delta + q0 + 8 * e + 4 * half);
#pragma unroll
        for (int f = 0; f < 4; ++f) p[4 * e + f] = -dl[f];
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = O::mma(Tl::row(at, 0, ks, lane_at), HELD ? k[HELD ? ks : 0] : Tl::row(my_k, 0, ks, lane_at), s);
        p = O::mma(Tl::row(at + BLOCK, 0, ks, lane_at), HELD ? v[HELD ? ks : 0] : Tl::row(my_k + BLOCK, 0, ks, lane_at), p);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 ls = *(LdsFour*)(s_lse + q0 + 8 * e + 4 * half);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          s[4 * e + f] = fast_exp2(fmaf(s[4 * e + f], a.c, -ls[f]));
          p[4 * e + f] = s[4 * e + f] * unit.times(p[4 * e + f]);
        }
      }
      if (q0 < all || q0 + 32 > nq) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int i = q0 + 8 * (e >> 2) + 4 * half + (e & 3);
          const bool in = i >= seen && i < nq;
          s[e] = in ? s[e] : 0.f;
          p[e] = in ? p[e] : 0.f;
        }
      }
      unit.fit(p, [&](float f) { scale_all(ak, f); });
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const Frag fp = O::pack(s, x), fs = O::pack(p, x);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          av[db] = O::mma(Tl::col(at + BLOCK, 16 * x, db, lane_at), fp, av[db]);
          ak[db] = O::mma(Tl::col(at, 16 * x, db, lane_at), fs, ak[db]);
        }
      }
    }
    if constexpr (O::F16) scale_all(ak, O::GRAD_UNIT * unit.back());
    if (a.causal && (any_nan<O>(ak) || any_nan<O>(av))) {
      // (delta of all queries is in LDS alone)
      float again[32 * DB];
      const Queries<T> s{(const T*)a.q.p + b * a.q.batch + (int64_t)h * a.q.head,
                         (const T*)a.g.p + b * a.g.batch + (int64_t)h * a.g.head,
                         a.q.token, 0, a.g.token, 0, lse + head0, (const float*)s_delta, a.queries, nq, INT_MAX, 0};
      strict_dkv<T, KS>((const T*)a.k.p + b * a.k.batch + (int64_t)key * a.k.token + (int64_t)h * a.k.head,
                        (const T*)a.v.p + b * a.v.batch + (int64_t)key * a.v.token + (int64_t)h * a.v.head, key < nk, s,
                        a.d, Range{begin / 32, (nq + 31) / 32, 1, 32}, seen, a.c, again);
      take<DB>(ak, again);
      take<DB>(av, again + 16 * DB);
    }
    if (first < a.keys) {
      if (key >= nk)
#pragma unroll
        for (int db = 0; db < DB; ++db) ak[db] = av[db] = zero16();
      // (this wave's keys and values are no longer read)
      store_rows<T, DB>(my_k, ak, a.scale, a.d, lane, to(dk, a.keys, a.key_heads));
      store_rows<T, DB>(my_k + BLOCK, av, O::GRAD_UNIT, a.d, lane, to(dv, a.keys, a.key_heads));
    }
  }
  if constexpr (!HELD) {
    if (dq) {
      __syncthreads();  // queries are no longer read
      if (first < a.queries) {
        packed.put(my_q, lane);
        Rows<T, DB>::flush(my_q, a.d, lane, to(dq, a.queries, a.heads));
      }
    }
  }
}

}  // namespace attn
}  // namespace mec
