// C-ABI entry points of attention (include/mec.h): argument validation in plain
// host code, then stream-ordered kernel launches.  Nothing here allocates device
// memory or synchronises the host.
#include <cmath>

#include "mec_attn_bwd.h"
#include "mec_attn_fwd.h"
#include "mec_heads.h"

using namespace mec;
using namespace mec::attn;

namespace {

constexpr int64_t kMaxRows = int64_t(1) << 30;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round256(int64_t b) { return (b + 255) & ~int64_t(255); }

int check_attention(const mec_attention_t* p, Problem* out) {
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
  if (p->keys > kMaxRows || p->queries > kMaxRows || group > kMaxRows || p->queries * group > kMaxRows ||
      p->batch > kMaxRows || p->key_heads > kMaxRows || p->batch * p->key_heads > kMaxRows)
    return fail(MEC_ERR_UNSUPPORTED, "%lld x %lld key heads, %lld queries for %lld heads each, %lld keys exceed 2^30",
                (long long)p->batch, (long long)p->key_heads, (long long)p->queries, (long long)group,
                (long long)p->keys);
  if (!(p->scale > 0.f && std::isfinite(p->scale))) return fail(MEC_ERR_INVALID, "scale must be finite and > 0");
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

View view(const mec_heads_t* h) { return View{h->data, h->batch_stride, h->token_stride, h->head_stride}; }

// A launch of `items` workgroups: a multiple of 8 ids over x and y.
struct Grid {
  int64_t items, ids;
  dim3 dims;
};
int make_grid(int64_t items, Grid* g) {
  g->items = items;
  g->ids = (items + 7) & ~int64_t(7);
  const int64_t x = g->ids < (1 << 20) ? g->ids : (1 << 20), y = ceil_div(g->ids, x);
  if (y > 65535) return fail(MEC_ERR_UNSUPPORTED, "%lld workgroups are too many", (long long)items);
  g->dims = dim3((unsigned)x, (unsigned)y);
  return MEC_OK;
}

// f(T*, integral_constant<KS>): KS steps of 16 features
template <class F>
void with_kernel(int dtype, int d, F f) {
  with_element_type(dtype, [&](auto* t) {
    if (d <= 32)
      f(t, std::integral_constant<int, 2>{});
    else if (d <= 64)
      f(t, std::integral_constant<int, 4>{});
    else if (d <= 80)
      f(t, std::integral_constant<int, 5>{});
    else if (d <= 96)
      f(t, std::integral_constant<int, 6>{});
    else
      f(t, std::integral_constant<int, 8>{});
  });
}

// How the forward's work is cut.
struct Plan {
  bool few;        // few rows a key head: the waves of a workgroup share them
  int row_tiles, splits;
  int64_t parts_o, parts_ml;  // bytes
};
constexpr int kWave = 4;

int plan_forward(const Problem& a, Plan* out) {
  const int64_t rows = (int64_t)a.queries * a.group;
  Plan p{};
  p.few = rows <= 32;
  p.row_tiles = (int)ceil_div(rows, p.few ? 32 : 128);
  p.splits = 1;
  if (p.few) {
    int cus = 0;
    if (int rc = compute_units(&cus)) return rc;
    // two workgroups a CU, and two tiles of 32 keys a wave
    const int64_t want = ceil_div(2 * cus, a.pairs * p.row_tiles), most = ceil_div(a.keys, 32 * kWave * 2);
    const int64_t s = want < most ? want : most;
    p.splits = (int)(s < 1 ? 1 : s);
  }
  if (p.splits > 1) {
    p.parts_o = round256(p.splits * a.pairs * rows * a.d * 4);
    p.parts_ml = p.splits * a.pairs * rows * 8;
  }
  *out = p;
  return MEC_OK;
}

}  // namespace

extern "C" {

int64_t mec_attention_workspace_bytes(const mec_attention_t* attention) {
  g_err.clear();
  Problem a{};
  Plan p{};
  int rc = check_attention(attention, &a);
  if (!rc) rc = plan_forward(a, &p);
  return rc ? rc : p.parts_o + p.parts_ml;
}

int mec_attention(const mec_attention_t* attention, const mec_heads_t* query, const mec_heads_t* key,
                  const mec_heads_t* value, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                  void* stream) {
  g_err.clear();
  Problem a{};
  Plan p{};
  Grid g{};
  int rc = check_attention(attention, &a);
  if (!rc) rc = check_heads(query, "query");
  if (!rc) rc = check_heads(key, "key");
  if (!rc) rc = check_heads(value, "value");
  if (!rc && !out) rc = fail(MEC_ERR_INVALID, "out must be non-null");
  if (!rc) rc = check_not_capturing(stream);
  if (!rc) rc = plan_forward(a, &p);
  if (!rc) rc = check_scratch(workspace, workspace_bytes, p.parts_o + p.parts_ml);
  if (!rc) rc = make_grid(a.pairs * p.row_tiles * p.splits, &g);
  if (rc) return rc;
  a.q = view(query);
  a.k = view(key);
  a.v = view(value);
  hipStream_t st = (hipStream_t)stream;
  const Parts parts{(float*)workspace, (float2*)((char*)workspace + p.parts_o)};
  with_kernel(attention->dtype, a.d, [&](auto* t, auto ks) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int KS = decltype(ks)::value;
    if (p.few) {
      k_attn_forward<T, KS, 1, kWave>
          <<<g.dims, 64 * kWave, 0, st>>>(a, g.items, g.ids, p.row_tiles, p.splits, (T*)out, lse, parts);
      if (p.splits > 1) {
        const int64_t rows = a.pairs * a.queries * a.group, groups = ceil_div(rows, 4);
        const int64_t x = groups < (1 << 20) ? groups : (1 << 20);
        k_attn_join<T><<<dim3((unsigned)x, (unsigned)ceil_div(groups, x)), 256, 0, st>>>(a, rows, p.splits, parts,
                                                                                        (T*)out, lse);
      }
    } else {
      k_attn_forward<T, KS, kWave, 1><<<g.dims, 64 * kWave, 0, st>>>(a, g.items, g.ids, p.row_tiles, 1, (T*)out, lse, parts);
    }
  });
  return check_launch("mec_attention");
}

int64_t mec_attention_backward_workspace_bytes(const mec_attention_t* attention) {
  g_err.clear();
  Problem a{};
  int rc = check_attention(attention, &a);
  return rc ? rc : a.pairs * a.queries * a.group * (int64_t)sizeof(float);
}

int mec_attention_backward(const mec_attention_t* attention, const mec_heads_t* query, const mec_heads_t* key,
                           const mec_heads_t* value, const void* out, const float* lse, const mec_heads_t* grad_out,
                           void* grad_query, void* grad_key, void* grad_value, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  g_err.clear();
  Problem a{};
  Grid gq{}, gk{};
  int rc = check_attention(attention, &a);
  if (!rc) rc = check_heads(query, "query");
  if (!rc) rc = check_heads(key, "key");
  if (!rc) rc = check_heads(value, "value");
  if (!rc) rc = check_heads(grad_out, "grad_out");
  if (!rc && (!out || !lse)) rc = fail(MEC_ERR_INVALID, "out and lse must be non-null");
  if (!rc && (!grad_key != !grad_value)) rc = fail(MEC_ERR_INVALID, "grad_key and grad_value go together");
  if (!rc) rc = check_scratch(workspace, workspace_bytes, a.pairs * a.queries * a.group * (int64_t)sizeof(float));
  if (!rc) rc = check_not_capturing(stream);
  const int64_t rows = (int64_t)a.queries * a.group;
  const int row_tiles = (int)ceil_div(rows, 128), key_tiles = (int)ceil_div(a.keys, 128);
  if (!rc) rc = make_grid(a.pairs * row_tiles, &gq);
  if (!rc) rc = make_grid(a.pairs * key_tiles, &gk);
  if (rc || (!grad_query && !grad_key)) return rc;
  a.q = view(query);
  a.k = view(key);
  a.v = view(value);
  a.g = view(grad_out);
  hipStream_t st = (hipStream_t)stream;
  float* delta = (float*)workspace;
  with_kernel(attention->dtype, a.d, [&](auto* t, auto ks) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int KS = decltype(ks)::value;
    k_attn_dq<T, KS><<<gq.dims, 256, 0, st>>>(a, gq.items, gq.ids, row_tiles, (const T*)out, lse, delta, (T*)grad_query);
    if (grad_key)
      k_attn_dkv<T, KS><<<gk.dims, 256, 0, st>>>(a, gk.items, gk.ids, key_tiles, lse, delta, (T*)grad_key,
                                                 (T*)grad_value);
  });
  return check_launch("mec_attention_backward");
}

}  // extern "C"
