// Attention's forward: one pass over the keys with the running maximum and sum
// of the softmax.
//
// The rows of a key head are its queries' heads, r = query * group + head: heads
// that share keys share the tiles read, and a single token's heads fill a wave.
// A wave holds 32 of them as right operands and forms S^T = K Q^T, 32 keys by 32
// rows, so that a lane's scores belong to one row; the maximum and the sum cross
// the lanes once a tile.  O^T = V^T P^T takes the probabilities from their lane.
// The maximum lags: the accumulators are rescaled only where it grew by more than
// 2^8, which after the first tiles hardly happens.
//
// WM > 1: WM waves of 32 rows each share tiles of KEYS keys, two in LDS, one of them
// on its way (Fetcher).  WM = 1 is the form for few rows (single tokens): the
// WK waves of a workgroup take every WK-th tile of 32 keys, each in LDS of its own
// without a barrier, and meet at the end; the keys are split over `splits`
// workgroups, which k_attn_join joins.
#pragma once
#include "mec_attn_strict.h"

namespace mec {
namespace attn {

// What a workgroup has of its rows where the keys are split: the sum of the values, and m (the maximum that it is
// relative to, in units of log2) and the sum of the probabilities.
struct Parts {
  float* o;    // [splits][pairs][rows][d]
  float2* ml;  // [splits][pairs][rows]
};

template <class T, int KS, int WM, int WK>
struct Forward {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  static constexpr int DB = (KS + 1) / 2;
  using Tl = Tile<T, DB>;
  static constexpr int NT = 64 * WM * WK, ROWS = 32 * WM;
  static constexpr int KEYS = WM == 1 || O::F32 ? 32 : 64, NB = KEYS / 32;
  static constexpr int TILE = KEYS * Tl::RB;
  // keys and values of a tile of each wave that has its own, and in the end (WM = 1) what the waves have
  static constexpr int TILES = 2 * TILE * WK, JOIN = WM == 1 ? WK * 32 * (32 * DB + 2) * 4 : 0;
  static constexpr int LDS = TILES > JOIN ? TILES : JOIN;
  static_assert(WM == 1 || WK == 1, "");
};

template <class T, int KS, int WM, int WK>
__global__ __launch_bounds__(64 * WM * WK, sizeof(T) == 4 || (WM == 1 && KS == 8) ? 1 : 2) void k_attn_forward(
    Problem a, Items items, int row_tiles, int splits, T* out, float* lse, Parts parts) {
  using F = Forward<T, KS, WM, WK>;
  using O = Ops<T>;
  using Frag = typename O::Frag;
  using Tl = typename F::Tl;
  constexpr int DB = F::DB, NB = F::NB, KEYS = F::KEYS;
  __shared__ alignas(16) char s_lds[F::LDS], s_next[WM == 1 ? 16 : F::LDS];
  int64_t pair;
  int in;
  if (!items.take(a.pairs, row_tiles * splits, pair, in)) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const typename Tl::At lane_at(lane);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (the last rows, where causal those that see most, first)
  const int split = in % splits, tile = row_tiles - 1 - in / splits;
  const int64_t b = pair / a.key_heads;
  const int kh = (int)(pair - b * a.key_heads);
  const int nq = a.nq(b), nk = a.nk(b), shift = nk - nq;
  const int rows = a.queries * a.group;
  // this lane's row
  const int row0 = tile * F::ROWS, wave_row0 = row0 + (WM == 1 ? 0 : 32 * wave);
  const int row = wave_row0 + (lane & 31);
  const int qi = row / a.group, qh = kh * a.group + row % a.group;
  const bool live = qi < nq;
  // keys that any row of the workgroup sees, and those that all rows of the wave do
  const int last = min((row0 + F::ROWS - 1) / a.group, nq - 1);
  int end = row0 / a.group >= nq ? 0 : a.causal ? min(nk, last + shift + 1) : nk;
  if (end < 0) end = 0;
  const int all = a.causal ? min(nk, wave_row0 / a.group + shift + 1) : nk;
  const int wave_end = wave_row0 / a.group >= nq ? 0
                       : a.causal               ? min(nk, min((wave_row0 + 31) / a.group, nq - 1) + shift + 1)
                                                : nk;
  const int see = a.causal ? min(nk, qi + shift + 1) : nk;  // this row sees the keys below

  f32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = zero16();
  float m = -kInf, l = 0.f;

  // tiles of this workgroup, and of this wave among them
  int first = 0, tiles = (end + KEYS - 1) / KEYS;
  if (WM == 1) {
    const int each = (tiles + splits - 1) / splits;
    first = split * each;
    tiles = min(tiles, first + each);
    first += wave;
  }
  if (first < tiles) {
    Frag q[KS];
    {
      const T* p = (const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)qh * a.q.head;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = O::load_row(p, live, s, half, a.d);
    }
    const auto use = [&](Lds* tk, int i) {
      auto at = lane_at;
      at.again();
      Lds* const tv = tk + F::TILE;
      const int key0 = i * KEYS;
      if (key0 >= wave_end) return;
      f32x16 s[NB];
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        s[kb] = zero16();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[kb] = O::mma(Tl::row(tk, 32 * kb, ks, at), q[ks], s[kb]);
      }
      if (key0 + KEYS > all) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[kb][e] = key0 + 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3) < see ? s[kb][e] : -kInf;
      }
      grow<O>(s, a.c, m, l, o);
      const float ref = (m == -kInf ? 0.f : m) - O::BIAS;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[kb][e] = fast_exp2(fmaf(s[kb][e], a.c, -ref));
          l += s[kb][e];
        }
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Frag p = O::pack(s[kb], h);
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db] = O::mma(Tl::col(tv, 32 * kb + 16 * h, db, at), p, o[db]);
        }
    };
    if constexpr (WM == 1) {
      Loader<T, DB, KEYS, 64> lk, lv;
      lk.init(a.k, b, kh, a.d, lane);
      lv.init(a.v, b, kh, a.d, lane);
      lk.load(first * KEYS, nk - first * KEYS);
      lv.load(first * KEYS, nk - first * KEYS);
      Lds* const tk = (Lds*)s_lds + wave * 2 * F::TILE;
      for (int i = first; i < tiles; i += WK) {
        lk.store(tk);
        lv.store(tk + F::TILE);
        wave_sync();
        if (i + WK < tiles) {
          lk.load((i + WK) * KEYS, nk - (i + WK) * KEYS);
          lv.load((i + WK) * KEYS, nk - (i + WK) * KEYS);
        }
        use(tk, i);
      }
    } else {
      Fetcher<T, DB, KEYS, WM> fk, fv;
      fk.init(a.k, b, kh, a.d, wave, lane);
      fv.init(a.v, b, kh, a.d, wave, lane);
      walk_tiles(
          first, tiles,
          [&](int i, auto place) {
            Lds* const tk = (Lds*)(place ? s_next : s_lds);
            fk.load(tk, i * KEYS, nk - i * KEYS);
            fv.load(tk + F::TILE, i * KEYS, nk - i * KEYS);
          },
          [&](int i, auto place) { use((Lds*)(place ? s_next : s_lds), i); });
    }
  }
  if (a.causal && any_nan<O>(o)) {
    float again[16 * DB + 2];
    strict_forward<T, KS>((const T*)a.q.p + b * a.q.batch + (int64_t)qi * a.q.token + (int64_t)qh * a.q.head, live,
                          (const T*)a.k.p + b * a.k.batch + (int64_t)kh * a.k.head, a.k.token,
                          (const T*)a.v.p + b * a.v.batch + (int64_t)kh * a.v.head, a.v.token, a.d,
                          Range{first, tiles, WK, KEYS}, wave_end, see, a.c, again);
    take<DB>(o, again);
    m = again[16 * DB];
    l = again[16 * DB + 1];
  }
  l += other_half(l);
  if (!live || l == 0.f) {
    // a row without a query, or that sees nothing
    m = -kInf;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = zero16();
  }
  if constexpr (WM == 1) {
    // the waves' parts meet in LDS, each wave then has a share of the rows
    __syncthreads();
    float* const all_o = (float*)s_lds;                   // [WK][32 rows][32 DB]
    float2* const all_ml = (float2*)(all_o + WK * 32 * 32 * DB);  // [WK][32 rows]
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(f32x4*)(all_o + ((wave * 32 + (lane & 31)) * DB + db) * 32 + 8 * i + 4 * half) =
            f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
    if (half == 0) all_ml[wave * 32 + lane] = make_float2(m, l);
    __syncthreads();
    for (int r = wave; r < 32; r += WK) {
      const int rr = row0 + r;
      if (rr >= rows) break;
      float top = -kInf, sum = 0.f, w[WK];
#pragma unroll
      for (int i = 0; i < WK; ++i) top = fmaxf(top, all_ml[i * 32 + r].x);
#pragma unroll
      for (int i = 0; i < WK; ++i) {
        const float2 ml = all_ml[i * 32 + r];
        w[i] = ml.x == -kInf ? 0.f : fast_exp2(ml.x - top);
        sum += w[i] * ml.y;
      }
      const int ri = rr / a.group, rh = kh * a.group + rr % a.group;
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      for (int e = lane; e < a.d; e += 64) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < WK; ++i) v += w[i] * all_o[(i * 32 + r) * 32 * DB + e];
        if (splits > 1)
          parts.o[((split * a.pairs + pair) * rows + rr) * (int64_t)a.d + e] = v;
        else
          put(out + ((b * a.queries + ri) * a.heads + rh) * (int64_t)a.d + e, v * inv);
      }
      if (lane == 0) {
        if (splits > 1)
          parts.ml[(split * a.pairs + pair) * rows + rr] = make_float2(top, sum);
        else if (lse)
          lse[(b * a.heads + rh) * (int64_t)a.queries + ri] = sum == 0.f ? kInf : top - O::BIAS + log2f(sum);
      }
    }
  } else {
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    if (lse && half == 0 && row < rows)
      lse[(b * a.heads + qh) * (int64_t)a.queries + qi] = l == 0.f ? kInf : m - O::BIAS + log2f(l);
    Lds* const mine = wave_rows<KEYS, Tl::RB>(s_lds, s_next, wave);  // (the tiles are no longer read)
    store_rows<T, DB>(mine, o, inv, a.d, lane, [&](int r) -> T* {
      const int at = wave_row0 + r;
      return at < rows ? out + ((b * a.queries + at / a.group) * a.heads + kh * a.group + at % a.group) * (int64_t)a.d
                       : nullptr;
    });
  }
}

// Joins the parts of a row: a wave a row.
template <class T>
__global__ __launch_bounds__(256) void k_attn_join(Problem a, int64_t all_rows, int splits, Parts parts, T* out,
                                                   float* lse) {
  const int lane = threadIdx.x & 63;
  const int64_t at = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (at >= all_rows) return;
  const int rows = a.queries * a.group;
  const int64_t pair = at / rows, b = pair / a.key_heads;
  const int r = (int)(at - pair * rows), ri = r / a.group, rh = (int)(pair - b * a.key_heads) * a.group + r % a.group;
  float top = -kInf, sum = 0.f;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, parts.ml[s * all_rows + at].x);
  float v0 = 0.f, v1 = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float2 ml = parts.ml[s * all_rows + at];
    const float w = ml.x == -kInf ? 0.f : fast_exp2(ml.x - top);
    sum += w * ml.y;
    const float* o = parts.o + (s * all_rows + at) * a.d;
    if (lane < a.d) v0 += w * o[lane];
    if (lane + 64 < a.d) v1 += w * o[lane + 64];
  }
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  T* p = out + ((b * a.queries + ri) * a.heads + rh) * (int64_t)a.d;
  if (lane < a.d) put(p + lane, v0 * inv);
  if (lane + 64 < a.d) put(p + lane + 64, v1 * inv);
  if (lse && lane == 0)
    lse[(b * a.heads + rh) * (int64_t)a.queries + ri] = sum == 0.f ? kInf : top - Ops<T>::BIAS + log2f(sum);
}

}  // namespace attn
}  // namespace mec
