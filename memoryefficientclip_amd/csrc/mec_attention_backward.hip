// C-ABI entry points of attention's backward (include/mec.h): argument validation in
// plain host code, then stream-ordered kernel launches.  Nothing here allocates
// device memory or synchronises the host.
#include "mec_attn_bwd.h"
#include "mec_attn_whole.h"
#include "mec_attn_host.h"

using namespace mec;
using namespace mec::attn;

namespace {

// Waves and LDS of k_attn_whole_grad, 0 waves where it does not fit.  Where it does it was the faster form at all
// sizes, 2 to 256 x 12 heads (256 x 12 heads of 64, us, this form and two kernels that walk over tiles: 77 tokens 68
// and 131, 197 tokens 297 and 354, 257 tokens 414 and 571; fp32, 77 tokens, 395 and 459).
struct Whole {
  int waves;
  size_t lds;
};
Whole plan_whole(const Problem& a, int dtype) {
  const int size = dtype == MEC_DTYPE_F32 ? 4 : 2, steps = a.d <= 32 ? 2 : a.d <= 64 ? 4 : a.d <= 96 ? 6 : 8;
  const int row = 16 * steps * size, most = whole_waves(steps, size);
  const int64_t nq = (a.queries + 31) & ~31, nk = (a.keys + 31) & ~31;
  const int64_t lds = 2 * (nq + nk) * row + 8 * nq;
  const int blocks = (int)((nq > nk ? nq : nk) / 32);
  // (wider heads do not fit into the registers; queries leave through the place of keys and values)
  if (steps > whole_steps(size) || a.group != 1 || lds > kWholeLds || blocks > most || nq > 2 * nk) return {0, 0};
  return {blocks, (size_t)lds};
}

}  // namespace

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
  Grid gq{}, gk{}, gw{};
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
  if (!rc) rc = make_grid(a.pairs, &gw);
  if (rc || (!grad_query && !grad_key)) return rc;
  a.q = view(query);
  a.k = view(key);
  a.v = view(value);
  a.g = view(grad_out);
  hipStream_t st = (hipStream_t)stream;
  float* delta = (float*)workspace;
  const Whole whole = plan_whole(a, attention->dtype);
  with_kernel(attention->dtype, a.d, [&](auto* t, auto ks) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int KS = decltype(ks)::value;
    if constexpr (KS <= whole_steps(sizeof(T))) {
      if (whole.waves) {
        k_attn_whole_grad<T, KS><<<gw.dims, 64 * whole.waves, whole.lds, st>>>(
            a, gw.items, gw.ids, (const T*)out, lse, (T*)grad_query, (T*)grad_key, (T*)grad_value);
        return;
      }
    }
    k_attn_dq<T, KS><<<gq.dims, 256, 0, st>>>(a, gq.items, gq.ids, row_tiles, (const T*)out, lse, delta, (T*)grad_query);
    if (grad_key)
      k_attn_dkv<T, KS><<<gk.dims, 256, 0, st>>>(a, gk.items, gk.ids, key_tiles, lse, delta, (T*)grad_key,
                                                 (T*)grad_value);
  });
  return check_launch("mec_attention_backward");
}

}  // extern "C"
