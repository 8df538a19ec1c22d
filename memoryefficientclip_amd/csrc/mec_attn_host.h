// Host side shared by attention's forward and backward (include/mec.h).
#pragma once
#include <cmath>

#include "mec_attn.h"
#include "mec_heads.h"

namespace mec {
namespace attn {

constexpr int64_t kMaxLength = int64_t(1) << 30;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round256(int64_t b) { return (b + 255) & ~int64_t(255); }

inline int check_attention(const mec_attention_t* p, Problem* out) {
  if (p == nullptr) return fail(MEC_ERR_INVALID, "attention must be non-null");
  if (int rc = check_element_type(p->dtype)) return rc;
  if (p->batch < 1 || p->queries < 1 || p->keys < 1 || p->heads < 1 || p->key_heads < 1 || p->head_dim < 1)
    return fail(MEC_ERR_INVALID, "batch=%lld, queries=%lld, keys=%lld, heads=%lld, key_heads=%lld, head_dim=%lld must "
                "be >= 1", (long long)p->batch, (long long)p->queries, (long long)p->keys, (long long)p->heads,
                (long long)p->key_heads, (long long)p->head_dim);
  if (p->heads % p->key_heads != 0)
    return fail(MEC_ERR_INVALID, "key_heads=%lld must divide heads=%lld", (long long)p->key_heads, (long long)p->heads);
  if (p->head_dim > MEC_MAX_HEAD_DIM)
    return fail(MEC_ERR_UNSUPPORTED, "head_dim=%lld exceeds the maximum %d", (long long)p->head_dim, MEC_MAX_HEAD_DIM);
  const int64_t group = p->heads / p->key_heads;
  if (p->keys > kMaxLength || p->queries > kMaxLength || group > kMaxLength || p->queries * group > kMaxLength ||
      p->batch > kMaxLength || p->key_heads > kMaxLength || p->batch * p->key_heads > kMaxLength)
    return fail(MEC_ERR_UNSUPPORTED, "%lld x %lld key heads, %lld queries for %lld heads each, %lld keys exceed 2^30",
                (long long)p->batch, (long long)p->key_heads, (long long)p->queries, (long long)group,
                (long long)p->keys);
  // (times log2(e) it has to be finite, and times -inf to be -inf)
  if (!(p->scale >= 1e-30f && p->scale <= 1e30f)) return fail(MEC_ERR_INVALID, "scale must be in [1e-30, 1e30]");
  if ((p->query_lengths || p->key_lengths) && p->length_bytes != 4 && p->length_bytes != 8)
    return fail(MEC_ERR_INVALID, "length_bytes=%d must be 4 or 8", p->length_bytes);
  Problem a{};
  a.queries = (int)p->queries;
  a.keys = (int)p->keys;
  a.heads = (int)p->heads;
  a.key_heads = (int)p->key_heads;
  a.group = (int)group;
  a.d = (int)p->head_dim;
  a.pairs = p->batch * p->key_heads;
  a.causal = p->causal != 0;
  a.scale = p->scale;
  a.c = p->scale * kLog2e;
  a.query_lengths = p->query_lengths;
  a.key_lengths = p->key_lengths;
  a.length64 = p->length_bytes == 8;
  *out = a;
  return MEC_OK;
}

inline View view(const mec_heads_t* h) { return View{h->data, h->batch_stride, h->token_stride, h->head_stride}; }

// A launch of `count` workgroups.
struct Grid {
  Items items;
  dim3 dims;
};
inline int make_grid(int64_t count, Grid* g) {
  const int64_t ids = (count + 7) & ~int64_t(7), x = ids < (1 << 20) ? ids : (1 << 20), y = ceil_div(ids, x);
  if (y > 65535) return fail(MEC_ERR_UNSUPPORTED, "%lld workgroups are too many", (long long)count);
  g->items = {count, ids};
  g->dims = dim3((unsigned)x, (unsigned)y);
  return MEC_OK;
}

// f(integral_constant<KS>): KS steps of 16 features
template <class F>
void with_steps(int d, F f) {
  if (d <= 32)
    f(std::integral_constant<int, 2>{});
  else if (d <= 48)
    f(std::integral_constant<int, 3>{});
  else if (d <= 64)
    f(std::integral_constant<int, 4>{});
  else if (d <= 80)
    f(std::integral_constant<int, 5>{});
  else if (d <= 96)
    f(std::integral_constant<int, 6>{});
  else
    f(std::integral_constant<int, 8>{});
}
// f(T*, integral_constant<KS>)
template <class F>
void with_kernel(int dtype, int d, F f) {
  with_element_type(dtype, [&](auto* t) { with_steps(d, [&](auto ks) { f(t, ks); }); });
}

}  // namespace attn
}  // namespace mec
