// The launches of attention's backward (mec_attn_cut.h), instantiated by a source for each element type.
#pragma once
#include "mec_attn_bwd.h"
#include "mec_attn_cut.h"
#include "mec_attn_whole.h"

namespace mec {
namespace attn {

template <class T>
void launch_backward(const Launch& l) {
  const Problem& a = l.a;
  const Cut& c = l.cut;
  hipStream_t st = l.stream;
  T *dq = (T*)l.dq, *dk = (T*)l.dk, *dv = (T*)l.dv;
  with_steps(a.d, [&](auto ks) {
    constexpr int KS = decltype(ks)::value;
    if constexpr (KS <= whole_steps(sizeof(T))) {
      if (l.whole.waves) {
        k_attn_whole_grad<T, KS>
            <<<l.gq.dims, 64 * l.whole.waves, l.whole.lds, st>>>(a, l.gq.items, (const T*)l.out, l.lse, dq, dk, dv);
        return;
      }
    }
    if (c.few_rows)
      k_attn_dq<T, KS, 1><<<l.gq.dims, 256, 0, st>>>(a, l.gq.items, c.row_tiles, (const T*)l.out, l.lse, l.delta, dq);
    else
      k_attn_dq<T, KS, 4><<<l.gq.dims, 256, 0, st>>>(a, l.gq.items, c.row_tiles, (const T*)l.out, l.lse, l.delta, dq);
    if (!dk) return;
    if (c.few_keys)
      k_attn_dkv<T, KS, 1>
          <<<l.gk.dims, 256, 0, st>>>(a, l.gk.items, c.key_tiles, c.splits, l.lse, l.delta, dk, dv, l.parts);
    else
      k_attn_dkv<T, KS, 4>
          <<<l.gk.dims, 256, 0, st>>>(a, l.gk.items, c.key_tiles, c.splits, l.lse, l.delta, dk, dv, l.parts);
    if (l.parts) k_attn_dkv_join<T><<<l.gj.dims, 256, 0, st>>>(a, a.pairs * a.keys, c.splits, l.parts, dk, dv);
  });
}

}  // namespace attn
}  // namespace mec
