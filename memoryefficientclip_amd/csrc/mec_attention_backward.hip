// C-ABI entry points of attention's backward (include/mec.h): argument validation in
// plain host code, then stream-ordered kernel launches.  Nothing here allocates
// device memory or synchronises the host.
#include "mec_attn_cut.h"
#include "mec_attn_whole.h"

using namespace mec;
using namespace mec::attn;

namespace {

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

int plan_cut(const Problem& a, const Whole& whole, Cut* out) {
  Cut c{};
  int cus = 0;
  if (int rc = compute_units(&cus)) return rc;
  const int64_t rows = (int64_t)a.queries * a.group;
  c.splits = 1;
  if (!whole.waves) {
    c.few_rows = a.pairs * ceil_div(rows, 128) < cus;
    c.few_keys = a.pairs * ceil_div(a.keys, 128) < cus;
    c.row_tiles = (int)ceil_div(rows, c.few_rows ? 32 : 128);
    c.key_tiles = (int)ceil_div(a.keys, c.few_keys ? 32 : 128);
    c.delta = round256(a.pairs * rows * 4);
    // about 8 workgroups a CU, 8 tiles of queries or more each
    const int64_t want = 8 * cus / (a.pairs * c.key_tiles), most = a.group * ceil_div(a.queries, 64) / 8;
    const int64_t s = want < most ? want : most;
    c.splits = (int)(s < 1 ? 1 : s);
    if (c.splits > 1) c.parts = c.splits * a.pairs * a.keys * 2 * a.d * 4;
  }
  *out = c;
  return MEC_OK;
}

}  // namespace

extern "C" {

int64_t mec_attention_backward_workspace_bytes(const mec_attention_t* attention) {
  g_err.clear();
  Problem a{};
  Cut c{};
  int rc = check_attention(attention, &a);
  if (!rc) rc = plan_cut(a, plan_whole(a, attention->dtype), &c);
  return rc ? rc : c.delta + c.parts;
}

int mec_attention_backward(const mec_attention_t* attention, const mec_heads_t* query, const mec_heads_t* key,
                           const mec_heads_t* value, const void* out, const float* lse, const mec_heads_t* grad_out,
                           void* grad_query, void* grad_key, void* grad_value, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  g_err.clear();
  Problem a{};
  Whole whole{};
  Cut c{};
  Grid gq{}, gk{}, gj{};
  int rc = check_attention(attention, &a);
  if (!rc) rc = check_heads(query, "query");
  if (!rc) rc = check_heads(key, "key");
  if (!rc) rc = check_heads(value, "value");
  if (!rc) rc = check_heads(grad_out, "grad_out");
  if (!rc && (!out || !lse)) rc = fail(MEC_ERR_INVALID, "out and lse must be non-null");
  if (!rc && (!grad_key != !grad_value)) rc = fail(MEC_ERR_INVALID, "grad_key and grad_value go together");
  if (!rc) rc = check_not_capturing(stream);
  if (!rc) {
    whole = plan_whole(a, attention->dtype);
    rc = plan_cut(a, whole, &c);
  }
  if (!rc) rc = check_scratch(workspace, workspace_bytes, c.delta + c.parts);
  if (!rc) rc = make_grid(a.pairs * (whole.waves ? 1 : c.row_tiles), &gq);
  if (!rc && !whole.waves) rc = make_grid(a.pairs * c.key_tiles * c.splits, &gk);
  if (!rc && c.splits > 1) rc = make_grid(ceil_div(a.pairs * a.keys, 4), &gj);
  if (rc || (!grad_query && !grad_key)) return rc;
  a.q = view(query);
  a.k = view(key);
  a.v = view(value);
  a.g = view(grad_out);
  hipStream_t st = (hipStream_t)stream;
  float* delta = (float*)workspace;
  float* parts = c.splits > 1 ? (float*)((char*)workspace + c.delta) : nullptr;
  const Launch l{a, whole, c, gq, gk, gj, lse, delta, parts, out, grad_query, grad_key, grad_value, st};
  with_element_type(attention->dtype, [&](auto* t) { launch_backward<std::remove_pointer_t<decltype(t)>>(l); });
  return check_launch("mec_attention_backward");
}

}  // extern "C"
