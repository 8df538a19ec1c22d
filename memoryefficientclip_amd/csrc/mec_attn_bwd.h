// Attention's backward, which makes the probabilities anew from the scores and
// the forward's lse.
//
// Two kernels, neither with atomics: k_attn_dq walks over the keys for 32 rows a
// wave (three products: S, dP, dQ), k_attn_dkv over the queries of all heads that
// share a key head for 32 keys a wave (four: S, dP, dV, dK).  S and dP are made
// twice, seven products for the five that one kernel would need, which would have
// to add its dQ over the key tiles in memory: with atomics in no fixed order, or
// in a pass of its own.  Gradients of the scores are rounded to T like the results:
// in fp16, to steps of 2^-24 and up to 65504, as the gradients that go out are.
// k_attn_dq also leaves delta = do . o for k_attn_dkv.
#pragma once
#include <climits>

#include "mec_attn.h"

namespace mec {
namespace attn {

template <class T, int KS>
struct Backward {
  using O = Ops<T>;
  static constexpr int DB = (KS + 1) / 2, WAVES = 4, NT = 64 * WAVES, ROWS = 32 * WAVES;
  using Tl = Tile<T, DB>;
  // rows of the tiles that are walked over
  static constexpr int KEYS = O::F32 || DB > 3 ? 32 : 64, QUERIES = O::F32 || DB > 3 ? 32 : 64;
  // the values of a wave's keys stay in LDS where keys, values and both gradients take
  // more registers than two waves on a SIMD have
  static constexpr bool V_LDS = !O::F32 && DB > 3;
  // The forward's result has the errors of 16 bits, and so has do . o; where few keys share a row's weight
  // this is the largest error of dq and dk (heads of 64, 77 tokens, causal, bf16: 0.0031 of their size, 0.0023
  // with a delta of fp32).  delta is also sum_j p_ij do_i . v_j: with d for do . o, eps = sum_j p_ij (do_i . v_j - d)
  // is what it lacks.  Up to KEYS_EXACT keys it is summed along with dq, and dq corrected by -eps sum_j p_ij k_j
  // (its product costs no reads of LDS), or, where registers are short, summed in a first walk over the keys.
  static constexpr int KEYS_EXACT = O::F32 ? 0 : 512;
  static constexpr bool TWICE = DB > 2;
};

template <class T, int KS>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void k_attn_dq(Problem a, int64_t items, int64_t ids, int row_tiles, const T* out,
                                                 const float* lse, float* delta, T* dq) {
  using B = Backward<T, KS>;
  using O = Ops<T>;
  using Frag = typename O::Frag;
  using Tl = typename B::Tl;
  constexpr int DB = B::DB, KEYS = B::KEYS, NB = KEYS / 32, TILE = KEYS * Tl::RB;
  __shared__ alignas(16) char s_lds[4 * TILE];
  Lds* const lds = (Lds*)s_lds;
  const int64_t id = group_id(ids);
  if (id >= items) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t pair = id / row_tiles;
  const int tile = row_tiles - 1 - (int)(id - pair * row_tiles);
  const int64_t b = pair / a.key_heads;
  const int kh = (int)(pair - b * a.key_heads);
  const int nq = a.nq(b), nk = a.nk(b), shift = nk - nq;
  const int rows = a.queries * a.group;
  const int row0 = tile * B::ROWS, wave_row0 = row0 + 32 * wave;
  const int row = wave_row0 + (lane & 31);
  const int qi = row / a.group, qh = kh * a.group + row % a.group;
  const bool live = qi < nq;
  const int last = min((row0 + B::ROWS - 1) / a.group, nq - 1);
  int end = row0 / a.group >= nq ? 0 : a.causal ? min(nk, last + shift + 1) : nk;
  if (end < 0) end = 0;
  const bool exact = end <= B::KEYS_EXACT;
  if (dq == nullptr && !exact) end = 0;
  const int all = a.causal ? min(nk, wave_row0 / a.group + shift + 1) : nk;
  const int wave_end = wave_row0 / a.group >= nq ? 0
                       : a.causal               ? min(nk, min((wave_row0 + 31) / a.group, nq - 1) + shift + 1)
                                                : nk;
  const int see = a.causal ? min(nk, qi + shift + 1) : nk;

  const int64_t at = (b * a.heads + qh) * (int64_t)a.queries + qi;  // of lse and delta
  Frag q[KS], g[KS];
  float dot = 0.f, l2 = kInf;
  {
    const T* pg = (const T*)a.g.p + b * a.g.batch + (int64_t)qi * a.g.token + (int64_t)qh * a.g.head;
    const T* po = out + ((b * a.queries + qi) * a.heads + qh) * (int64_t)a.d;
    const T* pq = (const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)qh * a.q.head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      g[s] = O::load_row(pg, live, s, half, a.d);
      dot += O::dot(g[s], O::load_row(po, live, s, half, a.d));
      q[s] = O::load_row(pq, live, s, half, a.d);
    }
    dot += other_half(dot);
    if (live) l2 = lse[at];
  }
  f32x16 acc[DB], mean[B::TWICE ? 1 : DB];  // dq / scale, sum_j p_ij k_j
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    acc[db] = zero16();
    mean[B::TWICE ? 0 : db] = zero16();
  }
  float eps = 0.f;
  const int tiles = (end + KEYS - 1) / KEYS;
  if (tiles > 0) {
    Loader<T, DB, KEYS, B::NT> lk, lv;
    lk.init(a.k, b, kh, a.d, threadIdx.x);
    lv.init(a.v, b, kh, a.d, threadIdx.x);
    lk.load(0, nk);
    lv.load(0, nk);
    // (the first walk: below 0)
    for (int i = B::TWICE && exact ? -tiles : 0; i < tiles; ++i) {
      Lds* const tk = lds + (i & 1 ? 2 * TILE : 0);
      Lds* const tv = tk + TILE;
      lk.store(tk);
      lv.store(tv);
      __syncthreads();
      if (i + 1 < tiles) {
        const int next = (i + 1 < 0 ? i + 1 + tiles : i + 1) * KEYS;
        lk.load(next, nk - next);
        lv.load(next, nk - next);
      }
      if (B::TWICE && i == 0 && exact) {
        dot += eps + other_half(eps);
        eps = 0.f;
      }
      const int key0 = (i < 0 ? i + tiles : i) * KEYS;
      if (key0 >= wave_end) continue;
      const bool masked = key0 + KEYS > all;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        f32x16 s = zero16(), p = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s = O::mma(Tl::row(tk, 32 * kb, ks, lane), q[ks], s);
          p = O::mma(Tl::row(tv, 32 * kb, ks, lane), g[ks], p);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[e] = fast_exp2(fmaf(s[e], a.c, -l2));
          p[e] = s[e] * (p[e] - dot);
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool in = key0 + 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3) < see;
            s[e] = in ? s[e] : 0.f;
            p[e] = in ? p[e] : 0.f;
          }
        }
        if (!O::F32 && exact) {
#pragma unroll
          for (int e = 0; e < 16; ++e) eps += p[e];
          if (B::TWICE && i < 0) continue;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Frag ds = O::pack(p, h);
          if (!O::F32 && !B::TWICE && exact) {
            const Frag ps = O::pack(s, h);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const Frag kt = Tl::col(tk, 32 * kb + 16 * h, db, lane);
              acc[db] = O::mma(kt, ds, acc[db]);
              mean[db] = O::mma(kt, ps, mean[db]);
            }
          } else {
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = O::mma(Tl::col(tk, 32 * kb + 16 * h, db, lane), ds, acc[db]);
          }
        }
      }
    }
  }
  if (!O::F32 && !B::TWICE && exact) {
    eps += other_half(eps);
    dot += eps;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[db][e] -= eps * mean[db][e];
  }
  if (half == 0 && row < rows) delta[at] = dot;
  if (dq == nullptr) return;
  if (!live || l2 == kInf)
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = zero16();
  __syncthreads();  // (the tiles are no longer read)
  store_rows<T, DB>(lds + 32 * wave * Tl::RB, acc, a.scale, a.d, lane, [&](int r) -> T* {
    const int to = wave_row0 + r;
    return to < rows ? dq + ((b * a.queries + to / a.group) * a.heads + kh * a.group + to % a.group) * (int64_t)a.d
                     : nullptr;
  });
}

template <class T, int KS>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void k_attn_dkv(Problem a, int64_t items, int64_t ids, int key_tiles,
                                                  const float* lse, const float* delta, T* dk, T* dv) {
  using B = Backward<T, KS>;
  using O = Ops<T>;
  using Frag = typename O::Frag;
  using Tl = typename B::Tl;
  constexpr int DB = B::DB, QUERIES = B::QUERIES, NB = QUERIES / 32, TILE = QUERIES * Tl::RB;
  __shared__ alignas(16) char s_lds[4 * TILE + (B::V_LDS ? B::ROWS * Tl::RB : 0)];
  __shared__ alignas(16) float s_row[2][2][QUERIES];  // lse, delta of the tile's queries
  Lds* const lds = (Lds*)s_lds;
  const int64_t id = group_id(ids);
  if (id >= items) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t pair = id / key_tiles;
  const int tile = (int)(id - pair * key_tiles);  // (where causal, the first keys are seen by most queries)
  const int64_t b = pair / a.key_heads;
  const int kh = (int)(pair - b * a.key_heads);
  const int nq = a.nq(b), nk = a.nk(b), shift = nk - nq;
  const int key0 = tile * B::ROWS, wave_key0 = key0 + 32 * wave;
  const int key = wave_key0 + (lane & 31);
  const bool live = key < nk;
  // queries that see any key of the workgroup, of the wave; those from which on all see all of the wave's; and
  // those from which on this key is seen
  const int begin = key0 >= nk ? nq : a.causal ? max(0, key0 - shift) : 0;
  const int wave_begin = wave_key0 >= nk ? INT_MAX : a.causal ? wave_key0 - shift : 0;
  const int all = a.causal ? wave_key0 + 31 - shift : 0;
  const int seen = a.causal ? key - shift : 0;

  f32x16 ak[DB], av[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) ak[db] = av[db] = zero16();
  const int first = begin / QUERIES, each = (nq + QUERIES - 1) / QUERIES - first;
  if (each > 0) {
    Frag k[KS], v[B::V_LDS ? 1 : KS];
    Lds* const values = lds + 4 * TILE;
    {
      const T* pk = (const T*)a.k.p + b * a.k.batch + (int64_t)key * a.k.token + (int64_t)kh * a.k.head;
      const T* pv = (const T*)a.v.p + b * a.v.batch + (int64_t)key * a.v.token + (int64_t)kh * a.v.head;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        k[s] = O::load_row(pk, live, s, half, a.d);
        const Frag x = O::load_row(pv, live, s, half, a.d);
        if constexpr (B::V_LDS)
          Tl::put_row(values, 32 * wave, s, lane, x);  // (read by this wave alone)
        else
          v[s] = x;
      }
    }
    Loader<T, DB, QUERIES, B::NT> lq, lg;
    float r_row = 0.f;  // threads below 2 QUERIES: a value of s_row on its way
    const int t = threadIdx.x;
    auto load = [&](int at) {
      const int h = kh * a.group + at / each, q0 = (first + at % each) * QUERIES;
      if (at % each == 0 || at == 0) {
        lq.init(a.q, b, h, a.d, t);
        lg.init(a.g, b, h, a.d, t);
      }
      lq.load(q0, nq - q0);
      lg.load(q0, nq - q0);
      if (t < 2 * QUERIES) {
        const int i = q0 + t % QUERIES;
        const float* p = (t < QUERIES ? lse : delta) + (b * a.heads + h) * (int64_t)a.queries;
        const float x = i < nq ? p[i] : t < QUERIES ? kInf : 0.f;
        r_row = t < QUERIES ? x - O::GRAD_BIAS : x * O::GRAD_UNIT;
      }
    };
    load(0);
    const int tiles = each * a.group;
    for (int i = 0; i < tiles; ++i) {
      Lds* const tq = lds + (i & 1 ? 2 * TILE : 0);
      Lds* const tg = tq + TILE;
      lq.store(tq);
      lg.store(tg);
      if (t < 2 * QUERIES) s_row[i & 1][t / QUERIES][t % QUERIES] = r_row;
      __syncthreads();
      if (i + 1 < tiles) load(i + 1);
      const int q0 = (first + i % each) * QUERIES;
      if (q0 + QUERIES <= wave_begin) continue;
      const bool masked = q0 < all;
#pragma unroll
      for (int qb = 0; qb < NB; ++qb) {
        f32x16 s = zero16(), p = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s = O::mma(Tl::row(tq, 32 * qb, ks, lane), k[ks], s);
          if constexpr (B::V_LDS)
            p = O::mma(Tl::row(tg, 32 * qb, ks, lane), Tl::row(values, 32 * wave, ks, lane), p);
          else
            p = O::mma(Tl::row(tg, 32 * qb, ks, lane), v[ks], p);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4 l2 = *(const f32x4*)&s_row[i & 1][0][32 * qb + 8 * e + 4 * half];
          const f32x4 dl = *(const f32x4*)&s_row[i & 1][1][32 * qb + 8 * e + 4 * half];
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            s[4 * e + f] = fast_exp2(fmaf(s[4 * e + f], a.c, -l2[f]));
            p[4 * e + f] = s[4 * e + f] * fmaf(p[4 * e + f], O::GRAD_UNIT, -dl[f]);
          }
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool in = q0 + 32 * qb + 8 * (e >> 2) + 4 * half + (e & 3) >= seen;
            s[e] = in ? s[e] : 0.f;
            p[e] = in ? p[e] : 0.f;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Frag fp = O::pack(s, h), fs = O::pack(p, h);
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            av[db] = O::mma(Tl::col(tg, 32 * qb + 16 * h, db, lane), fp, av[db]);
            ak[db] = O::mma(Tl::col(tq, 32 * qb + 16 * h, db, lane), fs, ak[db]);
          }
        }
      }
    }
  }
  if (!live)
#pragma unroll
    for (int db = 0; db < DB; ++db) ak[db] = av[db] = zero16();
  __syncthreads();  // (the tiles are no longer read)
  const auto to = [&](T* p) {
    return [&, p](int r) -> T* {
      return wave_key0 + r < a.keys ? p + ((b * a.keys + wave_key0 + r) * a.key_heads + kh) * (int64_t)a.d : nullptr;
    };
  };
  store_rows<T, DB>(lds + 32 * wave * Tl::RB, ak, a.scale, a.d, lane, to(dk));
  wave_sync();
  store_rows<T, DB>(lds + 32 * wave * Tl::RB, av, O::GRAD_UNIT, a.d, lane, to(dv));
}

}  // namespace attn
}  // namespace mec
