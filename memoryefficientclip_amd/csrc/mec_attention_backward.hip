// C-ABI entry points of attention's backward (include/mec.h): argument validation in
// plain host code, then stream-ordered kernel launches.  Nothing here allocates
// device memory or synchronises the host.
#include "mec_attn_bwd.h"
#include "mec_attn_host.h"

using namespace mec;
using namespace mec::attn;

extern "C" {

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
