// Attention's backward, which makes the probabilities anew from the scores and
// the forward's lse.
//
// Two kernels, neither with atomics: k_attn_dq walks over the keys for 32 rows a
// wave (three products: S, dP, dQ), k_attn_dkv over the queries of all heads that
// share a key head for 32 keys a wave (four: S, dP, dV, dK).  S and dP are made
// twice, seven products for the five that one kernel would need, which would have
// to add its dQ over the key tiles in memory: with atomics in no fixed order, or
// in a pass of its own.  Gradients of the scores are rounded to T (the MFMA's operand);
// in fp16 in units of their own (GradUnit).
// k_attn_dq also leaves delta = do . o for k_attn_dkv, and what that lacks where it
// has it (Backward), from a first walk of two products, or along with the mean key.
//
// WM = 4: the four waves of a workgroup have 32 rows (keys) each and share tiles,
// two in LDS, one of them on its way (Fetcher).  WM = 1, where that would leave the
// device empty: they share 32 rows (keys) and take every fourth tile of 32, each in
// LDS of its own, and add up what they have in the end.  k_attn_dkv's queries are
// split over `splits` workgroups besides, whose fp32 sums k_attn_dkv_join adds, where
// there are few keys, or the first ones are seen by many more queries than the last.
#pragma once
#include <climits>

#include "mec_attn_strict.h"

namespace mec {
namespace attn {

template <class T, int KS, int WM>
struct Backward {
  using O = Ops<T>;
  static constexpr int DB = (KS + 1) / 2, WAVES = 4, NT = 64 * WAVES, WK = WAVES / WM, ROWS = 32 * WM;
  static_assert(WM == 1 || WM == 4, "");
  using Tl = Tile<T, DB>;
  // rows of the tiles that are walked over
  static constexpr int STEP = WM == 1 || O::F32 || DB > 3 ? 32 : 64;
  static constexpr int TILE = STEP * Tl::RB;
  static constexpr int PLACE = 2 * TILE * WK;  // of a tile of each wave that has its own; WM = 4: there are two
  // (what leaves passes through the same LDS)
  static_assert(WM == 4 || WK * 32 * 32 * DB * 4 <= PLACE, "");
  // the values of a wave's keys, or the result's gradients of its rows, stay in LDS where
  // all that a wave holds takes more registers than two waves on a SIMD have
  static constexpr bool V_LDS = !O::F32 && DB > 3;
  // The forward's result has the errors of 16 bits, and so has do . o; where few keys share a row's weight
  // this is the largest error of dq and dk (heads of 64, 77 tokens, causal, bf16: 0.0031 of their size, 0.0023
  // with a delta of fp32).  delta is also sum_j p_ij do_i . v_j: with d for do . o, eps = sum_j p_ij (do_i . v_j - d)
  // is what it lacks.  Up to this many keys it is summed in a first walk over them.  Beyond, it would be two products on
  // three, and is left out: dq and dk, off by 0.60 of half a step in the mean square, are off by 0.75 where few of
  // 900 keys share a row's weight, and by 1.7 and 0.9 where the values have 4 times as much in common as they differ.
  //
  // dq = scale sum_j ds_ij k_j, and as the ds_ij add up to 0, the k_j might be less their mean, m_i = sum_j p_ij k_j:
  // rounded ds_ij do not add up to 0, and their sum times m_i is an error that grows with scale.  Heads of up to 48
  // have the registers for m_i: there dq is corrected by it, which takes what delta lacks along, at all lengths
  // (bf16, heads of 32, 6396 keys: dq off by 0.0026 of its size, 0.0023 with it; heads of 16: 0.0027 and 0.0023).
  // Wider heads over tiles do without: with keys that have 4 times as much in common as they differ dq is off by 1.8 to
  // 2.2 of half a step in the mean square, where it is 0.58 with the correction.
  static constexpr bool MEAN = !O::F32 && KS <= 3;
  static constexpr int KEYS_EXACT = O::F32 || MEAN ? -1 : 512;
};

// A row of the sums of a workgroup's waves, [WK][32][32 DB] in LDS.
template <int WK, int DB>
__device__ __forceinline__ float joined(const float* sums, int r, int e) {
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < WK; ++i) v += sums[(i * 32 + r) * 32 * DB + e];
  return v;
}
template <int DB>
__device__ __forceinline__ void put_sums(float* sums, const f32x16 (&acc)[DB], int wave, int lane) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(f32x4*)(sums + ((wave * 32 + (lane & 31)) * DB + db) * 32 + 8 * i + 4 * (lane >> 5)) =
          f32x4{acc[db][4 * i], acc[db][4 * i + 1], acc[db][4 * i + 2], acc[db][4 * i + 3]};
}

template <class T, int KS, int WM>
__global__ __launch_bounds__(256, sizeof(T) == 4 || (WM == 1 && KS > 4) ? 1 : 2) void k_attn_dq(
    Problem a, Items items, int row_tiles, const T* out, const float* lse, float* delta, T* dq) {
  using B = Backward<T, KS, WM>;
  using O = Ops<T>;
  using Frag = typename O::Frag;
  using Tl = typename B::Tl;
  constexpr int DB = B::DB, STEP = B::STEP, NB = STEP / 32, WK = B::WK;
  __shared__ alignas(16) char s_lds[B::PLACE], s_next[WM == 1 ? 16 : B::PLACE];
  __shared__ float s_eps[WM == 1 ? 2 * WK : 1][32];
  constexpr bool G_LDS = B::V_LDS && WM > 1;
  __shared__ alignas(16) char s_grads[G_LDS ? B::ROWS * Tl::RB : 16];
  int64_t pair;
  int tile;
  if (!items.take(a.pairs, row_tiles, pair, tile)) return;
  tile = row_tiles - 1 - tile;  // (where causal, the last rows see most keys)
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const typename Tl::At lane_at(lane);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = pair / a.key_heads;
  const int kh = (int)(pair - b * a.key_heads);
  const int nq = a.nq(b), nk = a.nk(b), shift = nk - nq;
  const int rows = a.queries * a.group;
  const int row0 = tile * B::ROWS, wave_row0 = row0 + (WM == 1 ? 0 : 32 * wave);
  const int row = wave_row0 + (lane & 31);
  const int qi = row / a.group, qh = kh * a.group + row % a.group;
  const bool live = qi < nq;
  const int last = min((row0 + B::ROWS - 1) / a.group, nq - 1);
  int end = row0 / a.group >= nq ? 0 : a.causal ? min(nk, last + shift + 1) : nk;
  if (end < 0) end = 0;
  const bool exact = end <= B::KEYS_EXACT;
  if (dq == nullptr && !exact && !B::MEAN) end = 0;
  const int all = a.causal ? min(nk, wave_row0 / a.group + shift + 1) : nk;
  const int wave_end = wave_row0 / a.group >= nq ? 0
                       : a.causal               ? min(nk, min((wave_row0 + 31) / a.group, nq - 1) + shift + 1)
                                                : nk;
  const int see = a.causal ? min(nk, qi + shift + 1) : nk;

  const int64_t at = (b * a.heads + qh) * (int64_t)a.queries + qi;  // of lse and delta
  Frag q[KS], g[G_LDS ? 1 : KS];
  Lds* const grads = (Lds*)s_grads + 32 * wave * Tl::RB;
  float dot = 0.f, l2 = kInf;
  {
    const T* pg = (const T*)a.g.p + b * a.g.batch + (int64_t)qi * a.g.token + (int64_t)qh * a.g.head;
    const T* po = out + ((b * a.queries + qi) * a.heads + qh) * (int64_t)a.d;
    const T* pq = (const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)qh * a.q.head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const Frag x = O::load_row(pg, live, s, half, a.d);
      dot += O::dot(x, O::load_row(po, live, s, half, a.d));
      if constexpr (G_LDS)
        Tl::put_row(grads, 0, s, lane, x);  // (read by this wave alone)
      else
        g[s] = x;
      q[s] = O::load_row(pq, live, s, half, a.d);
    }
    dot += other_half(dot);
    if (live) l2 = lse[at];
  }
  f32x16 acc[DB], mean[B::MEAN ? DB : 1];  // dq / scale; sum_j p_ij k_j
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    acc[db] = zero16();
    mean[B::MEAN ? db : 0] = zero16();
  }
  float eps = 0.f, eps16 = 0.f;  // sums of the ds_ij, and of the rounded ones
  GradUnit<O> unit;              // of them and of acc
  const int tiles = (end + STEP - 1) / STEP;
  if (tiles > 0) {
    const int first = WM == 1 ? wave : 0;
    int walk = exact ? 0 : 1;
    const auto use = [&](Lds* tk, int i) {
      auto at = lane_at;
      at.again();
      Lds* const tv = tk + B::TILE;
      const int key0 = i * STEP;
      if (key0 >= wave_end) return;
      const bool masked = key0 + STEP > all;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        f32x16 s = zero16(), p = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s = O::mma(Tl::row(tk, 32 * kb, ks, at), q[ks], s);
          if constexpr (G_LDS)
            p = O::mma(Tl::row(tv, 32 * kb, ks, at), Tl::row(grads, 0, ks, at), p);
          else
            p = O::mma(Tl::row(tv, 32 * kb, ks, at), g[ks], p);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[e] = fast_exp2(fmaf(s[e], a.c, -l2));
          p[e] = s[e] * unit.times(p[e], dot);
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool in = key0 + 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3) < see;
            s[e] = in ? s[e] : 0.f;
            p[e] = in ? p[e] : 0.f;
          }
        }
        unit.fit(p, [&](float f) {
          scale_all(acc, f);
          eps *= f;
          eps16 *= f;
        });
        if constexpr (B::MEAN) {
#pragma unroll
          for (int e = 0; e < 16; ++e) eps += p[e];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const Frag ds = O::pack(p, h), ps = O::pack(s, h);
            eps16 = O::add(ds, eps16);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const Frag kt = Tl::col(tk, 32 * kb + 16 * h, db, at);
              acc[db] = O::mma(kt, ds, acc[db]);
              mean[db] = O::mma(kt, ps, mean[db]);
            }
          }
          continue;
        }
        if constexpr (!O::F32) {
          // (one loop for both walks: the compiler's two copies of it take 50 registers more)
          int w = walk;
          asm volatile("" : "+v"(w));
          if (__builtin_amdgcn_readfirstlane(w) == 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) eps += p[e];
            continue;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Frag ds = O::pack(p, h);
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[db] = O::mma(Tl::col(tk, 32 * kb + 16 * h, db, at), ds, acc[db]);
        }
      }
    };
    Loader<T, DB, STEP, 64> lk, lv;
    Fetcher<T, DB, STEP, WM> fk, fv;
    if constexpr (WM == 1) {
      lk.init(a.k, b, kh, a.d, lane);
      lv.init(a.v, b, kh, a.d, lane);
    } else {
      fk.init(a.k, b, kh, a.d, wave, lane);
      fv.init(a.v, b, kh, a.d, wave, lane);
    }
#pragma unroll 1
    for (; walk < 2; ++walk) {
      if constexpr (WM == 1) {
        Lds* const tk = (Lds*)s_lds + wave * 2 * B::TILE;
        if (first < tiles) {
          lk.load(first * STEP, nk - first * STEP);
          lv.load(first * STEP, nk - first * STEP);
        }
        for (int i = first; i < tiles; i += WK) {
          lk.store(tk);
          lv.store(tk + B::TILE);
          wave_sync();
          if (i + WK < tiles) {
            lk.load((i + WK) * STEP, nk - (i + WK) * STEP);
            lv.load((i + WK) * STEP, nk - (i + WK) * STEP);
          }
          use(tk, i);
        }
      } else {
        walk_tiles(
            first, tiles,
            [&](int i, auto place) {
              Lds* const tk = (Lds*)(place ? s_next : s_lds);
              fk.load(tk, i * STEP, nk - i * STEP);
              fv.load(tk + B::TILE, i * STEP, nk - i * STEP);
            },
            [&](int i, auto place) { use((Lds*)(place ? s_next : s_lds), i); });
      }
      if (walk == 0) {
        if constexpr (O::F16) eps *= unit.back();
        eps += other_half(eps);
        if constexpr (WM == 1) {
          if (half == 0) s_eps[wave][lane] = eps;
          __syncthreads();
          eps = 0.f;
#pragma unroll
          for (int i = 0; i < WK; ++i) eps += s_eps[i][lane & 31];
        }
        dot += eps;
        eps = 0.f;
      }
    }
  }
  if constexpr (O::F16) {
    scale_all(acc, unit.back());
    eps *= unit.back();
    eps16 *= unit.back();
  }
  if constexpr (B::MEAN) {
    eps += other_half(eps);
    eps16 += other_half(eps16);
    if constexpr (WM == 1) {
      // (each wave takes its share of the correction off: the sum of all times its part of the mean)
      if (half == 0) {
        s_eps[wave][lane] = eps;
        s_eps[WK + wave][lane] = eps16;
      }
      __syncthreads();
      eps = eps16 = 0.f;
#pragma unroll
      for (int i = 0; i < WK; ++i) {
        eps += s_eps[i][lane & 31];
        eps16 += s_eps[WK + i][lane & 31];
      }
    }
    dot += eps;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[db][e] -= eps16 * mean[B::MEAN ? db : 0][e];
  }
  if (a.causal && any_nan<O>(acc)) {
    float again[16 * DB];
    strict_dq<T, KS>((const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)qh * a.q.head,
                     (const T*)a.g.p + b * a.g.batch + (int64_t)qi * a.g.token + (int64_t)qh * a.g.head, live,
                     (const T*)a.k.p + b * a.k.batch + (int64_t)kh * a.k.head, a.k.token,
                     (const T*)a.v.p + b * a.v.batch + (int64_t)kh * a.v.head, a.v.token, a.d,
                     Range{WM == 1 ? wave : 0, tiles, WK, STEP}, wave_end, see, a.c, l2, dot, again);
    take<DB>(acc, again);
  }
  if (half == 0 && row < rows && (WM > 1 || wave == 0)) delta[at] = dot;
  if (dq == nullptr) return;
  if (!live || l2 == kInf)
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = zero16();
  const auto to = [&](int r) -> T* {
    const int x = wave_row0 + r;
    return x < rows ? dq + ((b * a.queries + x / a.group) * a.heads + kh * a.group + x % a.group) * (int64_t)a.d : nullptr;
  };
  if constexpr (WM == 1) {
    __syncthreads();  // (the tiles are no longer read)
    put_sums<DB>((float*)s_lds, acc, wave, lane);
    __syncthreads();
    for (int r = wave; r < 32; r += WK)
      if (T* p = to(r))
        for (int e = lane; e < a.d; e += 64) put(p + e, a.scale * joined<WK, DB>((float*)s_lds, r, e));
  } else {
    store_rows<T, DB>(wave_rows<STEP, Tl::RB>(s_lds, s_next, wave), acc, a.scale, a.d, lane, to);
  }
}

template <class T, int KS, int WM>
__global__ __launch_bounds__(256, sizeof(T) == 4 || (WM == 1 && KS > 4) ? 1 : 2) void k_attn_dkv(
    Problem a, Items items, int key_tiles, int splits, const float* lse, const float* delta, T* dk, T* dv, float* parts) {
  using B = Backward<T, KS, WM>;
  using O = Ops<T>;
  using Frag = typename O::Frag;
  using Tl = typename B::Tl;
  constexpr int DB = B::DB, STEP = B::STEP, NB = STEP / 32, WK = B::WK;
  __shared__ alignas(16) char s_lds[B::PLACE], s_next[WM == 1 ? 16 : B::PLACE];
  __shared__ alignas(16) char s_values[B::V_LDS ? B::ROWS * Tl::RB : 16];
  // lse and delta of the tile's queries
  __shared__ alignas(16) float s_row[WK][2][64], s_next_row[2][64];
  int64_t pair;
  int tile;  // (where causal, the first keys are seen by most queries)
  if (!items.take(a.pairs, key_tiles * splits, pair, tile)) return;
  const int split = tile % splits;
  tile /= splits;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const typename Tl::At lane_at(lane);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = pair / a.key_heads;
  const int kh = (int)(pair - b * a.key_heads);
  const int nq = a.nq(b), nk = a.nk(b), shift = nk - nq;
  const int key0 = tile * B::ROWS, wave_key0 = key0 + (WM == 1 ? 0 : 32 * wave);
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
  GradUnit<O> unit(O::GRAD_UNIT);  // of ak, beside that of the probabilities
  // the tiles of all heads, and this workgroup's share of them
  const int first = begin / STEP, each = (nq + STEP - 1) / STEP - first;
  const int tiles = each > 0 ? each * a.group : 0, share = (tiles + splits - 1) / splits;
  const int stop = min(tiles, (split + 1) * share);
  if (split * share < stop) {
    Frag k[KS], v[B::V_LDS ? 1 : KS];
    Lds* const values = (Lds*)s_values + (WM == 1 ? 0 : 32 * wave * Tl::RB);
    if constexpr (WM == 4 && STEP == 64) {
      // (through the tiles' places, in whole rows, not as fragments, 16 bytes of each of 32 rows at a time: one query of
      // 729 keys, 256 x 16 heads of 72, 527 to 511 us)
      Fetcher<T, DB, 128, WM> fk, fv;
      fk.init(a.k, b, kh, a.d, wave, lane);
      fv.init(a.v, b, kh, a.d, wave, lane);
      fk.load((Lds*)s_lds, key0, nk - key0);
      fv.load((Lds*)s_next, key0, nk - key0);
      loads_done();
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        k[s] = Tl::row((Lds*)s_lds, 32 * wave, s, lane_at);
        v[s] = Tl::row((Lds*)s_next, 32 * wave, s, lane_at);
      }
      __syncthreads();
    } else {
      const T* pk = (const T*)a.k.p + b * a.k.batch + (int64_t)key * a.k.token + (int64_t)kh * a.k.head;
      const T* pv = (const T*)a.v.p + b * a.v.batch + (int64_t)key * a.v.token + (int64_t)kh * a.v.head;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        k[s] = O::load_row(pk, live, s, half, a.d);
        const Frag x = O::load_row(pv, live, s, half, a.d);
        if constexpr (B::V_LDS) {
          // (WM = 4: read by this wave alone; WM = 1: by all, which write the same)
          Tl::put_row(values, 0, s, lane, x);
        } else {
          v[s] = x;
        }
      }
    }
    const auto use = [&](Lds* tq, const float* row, int i) {
      auto at = lane_at;
      at.again();
      Lds* const tg = tq + B::TILE;
      const int q0 = (first + i % each) * STEP;
      if (q0 + STEP <= wave_begin) return;
      // (of rows beyond the queries Q and dO are 0, but 0 times a key that holds an inf is NaN)
      const bool masked = q0 < all || q0 + STEP > nq;
#pragma unroll
      for (int qb = 0; qb < NB; ++qb) {
        f32x16 s = zero16(), p = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s = O::mma(Tl::row(tq, 32 * qb, ks, at), k[ks], s);
          if constexpr (B::V_LDS)
            p = O::mma(Tl::row(tg, 32 * qb, ks, at), Tl::row(values, 0, ks, at), p);
          else
            p = O::mma(Tl::row(tg, 32 * qb, ks, at), v[ks], p);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4 l2 = *(const f32x4*)(row + 32 * qb + 8 * e + 4 * half);
          const f32x4 dl = *(const f32x4*)(row + 64 + 32 * qb + 8 * e + 4 * half);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            s[4 * e + f] = fast_exp2(fmaf(s[4 * e + f], a.c, O::GRAD_BIAS - l2[f]));
            p[4 * e + f] = s[4 * e + f] * unit.times(p[4 * e + f], dl[f]);
          }
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int i = q0 + 32 * qb + 8 * (e >> 2) + 4 * half + (e & 3);
            const bool in = i >= seen && i < nq;
            s[e] = in ? s[e] : 0.f;
            p[e] = in ? p[e] : 0.f;
          }
        }
        unit.fit(p, [&](float f) { scale_all(ak, f); });
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Frag fp = O::pack(s, h), fs = O::pack(p, h);
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            av[db] = O::mma(Tl::col(tg, 32 * qb + 16 * h, db, at), fp, av[db]);
            ak[db] = O::mma(Tl::col(tq, 32 * qb + 16 * h, db, at), fs, ak[db]);
          }
        }
      }
    };
    const int begin_at = split * share;
    if constexpr (WM == 1) {
      Loader<T, DB, STEP, 64> lq, lg;
      float r_row = 0.f;  // a query's lse or delta on its way
      const auto load = [&](int at) {
        const int h = kh * a.group + at / each, q0 = (first + at % each) * STEP;
        lq.init(a.q, b, h, a.d, lane);
        lg.init(a.g, b, h, a.d, lane);
        lq.load(q0, nq - q0);
        lg.load(q0, nq - q0);
        const int i = q0 + (lane & 31);
        // (of rows that are none Q and dO are 0)
        r_row = i < nq ? (half ? delta : lse)[(b * a.heads + h) * (int64_t)a.queries + i] : 0.f;
      };
      Lds* const tq = (Lds*)s_lds + wave * 2 * B::TILE;
      if (begin_at + wave < stop) load(begin_at + wave);
      for (int i = begin_at + wave; i < stop; i += WK) {
        lq.store(tq);
        lg.store(tq + B::TILE);
        s_row[wave][half][lane & 31] = r_row;
        wave_sync();
        if (i + WK < stop) load(i + WK);
        use(tq, s_row[wave][0], i);
      }
    } else {
      Fetcher<T, DB, STEP, WM> fq, fg;
      fq.init(a.q, b, kh * a.group, a.d, wave, lane, a.group > 1);
      fg.init(a.g, b, kh * a.group, a.d, wave, lane, a.group > 1);
      walk_tiles(
          begin_at, stop,
          [&](int at, auto place) {
            const int h = kh * a.group + at / each, q0 = (first + at % each) * STEP;
            fq.move(a.q, b, h);
            fg.move(a.g, b, h);
            Lds* const tq = (Lds*)(place ? s_next : s_lds);
            fq.load(tq, q0, nq - q0);
            fg.load(tq + B::TILE, q0, nq - q0);
            if (wave < 2) {
              // (lse by the first wave, delta by the second; of rows that are none 0, as their Q and dO)
              const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
                  (void*)((wave ? delta : lse) + (b * a.heads + h) * (int64_t)a.queries + q0), 0, 0x7fffffff, 0x00020000);
              Lds* const to = (Lds*)(place ? &s_next_row[0][0] : &s_row[0][0][0]) + wave * 256;
              __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)to, 4,
                                                       lane < STEP && q0 + lane < nq ? 4 * lane : OOB, 0, 0, 0);
            }
          },
          [&](int i, auto place) {
            use((Lds*)(place ? s_next : s_lds), place ? &s_next_row[0][0] : &s_row[0][0][0], i);
          });
    }
  }
  if constexpr (O::F16) scale_all(ak, O::GRAD_UNIT * unit.back());
  if (a.causal && (any_nan<O>(ak) || any_nan<O>(av))) {
    float again[32 * DB];
    const int h = kh * a.group;
    const int64_t head0 = (b * a.heads + h) * (int64_t)a.queries;
    const Queries<T> s{(const T*)a.q.p + b * a.q.batch + (int64_t)h * a.q.head,
                       (const T*)a.g.p + b * a.g.batch + (int64_t)h * a.g.head,
                       a.q.token, a.q.head, a.g.token, a.g.head, lse + head0, delta + head0, a.queries, nq, each, first};
    strict_dkv<T, KS>((const T*)a.k.p + b * a.k.batch + (int64_t)key * a.k.token + (int64_t)kh * a.k.head,
                      (const T*)a.v.p + b * a.v.batch + (int64_t)key * a.v.token + (int64_t)kh * a.v.head, live, s, a.d,
                      Range{split * share + (WM == 1 ? wave : 0), stop, WK, STEP}, seen, a.c, again);
    take<DB>(ak, again);
    take<DB>(av, again + 16 * DB);
  }
  if (!live)
#pragma unroll
    for (int db = 0; db < DB; ++db) ak[db] = av[db] = zero16();
  // where row r of dk or dv, or of a part's sums (dk's, then dv's d values), goes
  const auto to = [&](T* p) {
    return [&, p](int r) -> T* {
      return wave_key0 + r < a.keys ? p + ((b * a.keys + wave_key0 + r) * a.key_heads + kh) * (int64_t)a.d : nullptr;
    };
  };
  const auto part = [&](int r) -> float* {
    return wave_key0 + r < a.keys ? parts + ((split * a.pairs + pair) * a.keys + wave_key0 + r) * 2 * a.d : nullptr;
  };
  if constexpr (WM == 1) {
    __syncthreads();  // (the tiles are no longer read)
    float* const sums = (float*)s_lds;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      put_sums<DB>(sums, side ? av : ak, wave, lane);
      __syncthreads();
      for (int r = wave; r < 32; r += WK)
        if (wave_key0 + r < a.keys)
          for (int e = lane; e < a.d; e += 64) {
            const float x = joined<WK, DB>(sums, r, e);
            if (parts)
              part(r)[side * a.d + e] = x;
            else
              put((side ? to(dv) : to(dk))(r) + e, x * (side ? O::GRAD_UNIT : a.scale));
          }
      __syncthreads();
    }
  } else if (parts) {
    float* const p = part(lane & 31);
    if (p) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int x = 32 * db + 8 * (e >> 2) + 4 * half + (e & 3);
          if (x < a.d) {
            p[x] = ak[db][e];
            p[a.d + x] = av[db][e];
          }
        }
    }
  } else {
    Lds* const mine = wave_rows<STEP, Tl::RB>(s_lds, s_next, wave);
    store_rows<T, DB>(mine, ak, a.scale, a.d, lane, to(dk));
    wave_sync();
    store_rows<T, DB>(mine, av, O::GRAD_UNIT, a.d, lane, to(dv));
  }
}

// dk and dv from the parts' sums: a wave a key.
template <class T>
__global__ __launch_bounds__(256) void k_attn_dkv_join(Problem a, int64_t all_keys, int splits, const float* parts, T* dk,
                                                       T* dv) {
  const int64_t at = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (at >= all_keys) return;
  const int lane = threadIdx.x & 63;
  const int64_t pair = at / a.keys, b = pair / a.key_heads;
  const int key = (int)(at - pair * a.keys), kh = (int)(pair - b * a.key_heads);
  const int64_t to = ((b * a.keys + key) * a.key_heads + kh) * (int64_t)a.d;
  for (int e = lane; e < 2 * a.d; e += 64) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += parts[(s * all_keys + at) * 2 * a.d + e];
    if (e < a.d)
      put(dk + to + e, v * a.scale);
    else
      put(dv + to + e - a.d, v * Ops<T>::GRAD_UNIT);
  }
}

}  // namespace attn
}  // namespace mec
