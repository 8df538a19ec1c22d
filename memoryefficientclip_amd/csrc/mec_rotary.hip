// C-ABI entry points of the rotation of queries and keys (include/mec.h):
// argument validation in plain host code, then stream-ordered kernel launches.
// Nothing here allocates device memory or synchronises the host.
#include <cmath>

#include "mec_heads.h"
#include "mec_rotary.h"

using namespace mec;

namespace {

constexpr int64_t kMaxRotaryRows = int64_t(1) << 31, kMaxRotaryHeads = 1 << 16;

struct Rotary {
  RotaryShape s;
  int vp;  // pairs of a lane
};

int check_rotary(const mec_rotary_t* r, bool grad, Rotary* out) {
  if (r == nullptr) return fail(MEC_ERR_INVALID, "rotary must be non-null");
  if (int rc = check_element_type(r->dtype)) return rc;
  if (int rc = check_element_type(r->weight_dtype)) return rc;
  if (r->batch < 1 || r->tokens < 1 || r->query_heads < 0 || r->key_heads < 0 || r->query_heads + r->key_heads < 1)
    return fail(MEC_ERR_INVALID, "batch=%lld and tokens=%lld must be >= 1, query_heads=%lld and key_heads=%lld >= 0, not "
                "both 0", (long long)r->batch, (long long)r->tokens, (long long)r->query_heads, (long long)r->key_heads);
  if (r->head_dim < 2 || r->head_dim % 2 != 0)
    return fail(MEC_ERR_INVALID, "head_dim=%lld must be even and >= 2", (long long)r->head_dim);
  if (r->head_dim > 2 * kMaxHalf)
    return fail(MEC_ERR_UNSUPPORTED, "head_dim=%lld exceeds the maximum %d", (long long)r->head_dim, 2 * kMaxHalf);
  if (r->query_heads > kMaxRotaryHeads || r->key_heads > kMaxRotaryHeads || r->batch >= kMaxRotaryRows ||
      r->tokens >= kMaxRotaryRows || r->batch * r->tokens >= kMaxRotaryRows)
    return fail(MEC_ERR_UNSUPPORTED, "%lld x %lld tokens of %lld and %lld heads exceed the maxima 2^31 - 1 and 2^16",
                (long long)r->batch, (long long)r->tokens, (long long)r->query_heads, (long long)r->key_heads);
  if (r->axes < 1 || r->axes > MEC_MAX_AXES)
    return fail(MEC_ERR_INVALID, "axes=%d out of range [1, %d]", r->axes, MEC_MAX_AXES);
  RotaryShape s{};
  for (int a = 0; a < r->axes; ++a) {
    if (r->sections[a] < 0 || r->sections[a] > kMaxHalf)
      return fail(MEC_ERR_INVALID, "section %d of %d pairs out of range [0, %d]", a, r->sections[a], kMaxHalf);
    s.first[a + 1] = s.first[a] + r->sections[a];
  }
  s.half = (int)(r->head_dim / 2);
  if (s.first[r->axes] != s.half)
    return fail(MEC_ERR_INVALID, "the sections have %d pairs, a head of %lld features has %d", s.first[r->axes],
                (long long)r->head_dim, s.half);
  if (r->positions == nullptr) return fail(MEC_ERR_INVALID, "positions must be non-null");
  if (r->position_type < MEC_POSITION_INT32 || r->position_type > MEC_POSITION_F32)
    return fail(MEC_ERR_INVALID, "unknown position_type %d", r->position_type);
  if (!(r->theta > 0.0) || !std::isfinite(r->theta)) return fail(MEC_ERR_INVALID, "theta must be finite and > 0");
  if (r->norm && !(r->eps >= 0.f && std::isfinite(r->eps)))
    return fail(MEC_ERR_INVALID, "eps must be finite and >= 0");
  s.rows = r->batch * r->tokens;
  s.tokens = (int)r->tokens;
  s.heads[0] = (int)r->query_heads;
  s.heads[1] = (int)r->key_heads;
  // the waves of a workgroup, in proportion to the heads
  const int64_t all = r->query_heads + r->key_heads;
  s.waves[0] = (int)((kRotaryWaves * r->query_heads + all / 2) / all);
  if (r->query_heads && s.waves[0] < 1) s.waves[0] = 1;
  if (r->key_heads && s.waves[0] > kRotaryWaves - 1) s.waves[0] = kRotaryWaves - 1;
  s.waves[1] = kRotaryWaves - s.waves[0];
  s.axes = r->axes;
  s.pos = r->positions;
  s.pos_kind = r->position_type;
  s.pos_batch = r->positions_per_batch ? r->tokens * r->axes : 0;
  s.freq = r->frequencies;
  s.log2_theta = std::log2(r->theta);
  s.sign = 1.f;
  s.eps = r->eps;
  s.weight_dtype = r->weight_dtype;
  s.w[0] = r->norm ? r->query_weight : nullptr;
  s.w[1] = r->norm ? r->key_weight : nullptr;
  // Whole 16-byte vectors of pairs where they divide a half, else half vectors.  The norm's gradient holds too much of
  // each pair for 8 of them: 4 a lane took 0.39 ms for 128 x 1024 tokens of 24 heads of 64 in bf16, 8 a lane 0.45 ms
  // (4 x 32768 tokens, 40 heads of 128: 0.87 and 1.04 ms), the forward the other way round 0.27 and 0.22 ms.
  const int whole = r->dtype == MEC_DTYPE_F32 ? 4 : 8;
  out->vp = s.half % whole == 0 && !(grad && r->norm && whole == 8) ? whole : whole / 2;
  while (out->vp << s.lg < s.half) ++s.lg;
  out->s = s;
  return MEC_OK;
}

int check_sides(const Rotary& r, const mec_heads_t* q, const mec_heads_t* k, const char* what) {
  for (int e = 0; e < 2; ++e)
    if (r.s.heads[e])
      if (int rc = check_heads(e ? k : q, what)) return rc;
  return MEC_OK;
}

HeadsView view(const mec_heads_t* h) {
  return h ? HeadsView{h->data, h->batch_stride, h->token_stride, h->head_stride} : HeadsView{};
}

// A wave takes a side of a token at a time; workgroups enough for all, or to fill the device.
int rotary_groups(const Rotary& r, int per_cu, int* groups) {
  int cus = 0;
  if (int rc = compute_units(&cus)) return rc;
  int least = kRotaryWaves;
  for (int e = 0; e < 2; ++e)
    if (r.s.heads[e] && r.s.waves[e] < least) least = r.s.waves[e];
  const int64_t need = (r.s.rows + least - 1) / least, most = (int64_t)cus * per_cu;
  *groups = (int)(need < most ? need : most);
  return MEC_OK;
}

// f(T*, integral_constant<VP>, integral_constant<interleaved>)
template <class F>
void with_rotary(int dtype, int vp, int interleaved, F f) {
  with_element_type(dtype, [&](auto* t) {
    constexpr int N = 16 / sizeof(*t);
    auto go = [&](auto n) {
      if (interleaved)
        f(t, n, std::true_type{});
      else
        f(t, n, std::false_type{});
    };
    if (vp == N)
      go(std::integral_constant<int, N>{});
    else
      go(std::integral_constant<int, N / 2>{});
  });
}

constexpr int kForwardPerCu = 8, kGradPerCu = 4;

void launch_rotary(const Rotary& r, const mec_rotary_t* p, bool norm, const mec_heads_t* q, const mec_heads_t* k, void* yq,
                   void* yk, int groups, hipStream_t st) {
  with_rotary(p->dtype, r.vp, p->interleaved, [&](auto* t, auto vp, auto il) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int VP = decltype(vp)::value;
    constexpr bool IL = decltype(il)::value;
    if (norm)
      k_rotary<T, VP, IL, true><<<groups, 64 * kRotaryWaves, 0, st>>>(r.s, view(q), view(k), (T*)yq, (T*)yk);
    else
      k_rotary<T, VP, IL, false><<<groups, 64 * kRotaryWaves, 0, st>>>(r.s, view(q), view(k), (T*)yq, (T*)yk);
  });
}

}  // namespace

extern "C" {

int mec_norm_rotary(const mec_rotary_t* rotary, const mec_heads_t* query, const mec_heads_t* key, void* out_query,
                    void* out_key, void* stream) {
  g_err.clear();
  Rotary r{};
  int groups = 0;
  int rc = check_rotary(rotary, false, &r);
  if (!rc) rc = check_sides(r, query, key, "query and key");
  if (!rc && ((r.s.heads[0] && !out_query) || (r.s.heads[1] && !out_key)))
    rc = fail(MEC_ERR_INVALID, "out_query and out_key must be non-null");
  if (!rc) rc = check_not_capturing(stream);
  if (!rc) rc = rotary_groups(r, kForwardPerCu, &groups);
  if (rc) return rc;
  launch_rotary(r, rotary, rotary->norm, query, key, out_query, out_key, groups, (hipStream_t)stream);
  return check_launch("mec_norm_rotary");
}

int64_t mec_norm_rotary_workspace_bytes(const mec_rotary_t* rotary) {
  g_err.clear();
  Rotary r{};
  int groups = 0;
  int rc = check_rotary(rotary, true, &r);
  if (rc || !rotary->norm) return rc;
  rc = rotary_groups(r, kGradPerCu, &groups);
  return rc ? rc : (int64_t)groups * 4 * r.s.half * (int64_t)sizeof(float);
}

int mec_norm_rotary_backward(const mec_rotary_t* rotary, const mec_heads_t* query, const mec_heads_t* key,
                             const mec_heads_t* grad_out_query, const mec_heads_t* grad_out_key, void* grad_query,
                             void* grad_key, void* grad_query_weight, void* grad_key_weight, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  g_err.clear();
  Rotary r{};
  int groups = 0;
  int rc = check_rotary(rotary, true, &r);
  if (!rc) rc = check_sides(r, grad_out_query, grad_out_key, "grad_out_query and grad_out_key");
  if (!rc && rotary->norm) rc = check_sides(r, query, key, "query and key");
  if (!rc && !rotary->norm && (grad_query_weight || grad_key_weight))
    rc = fail(MEC_ERR_INVALID, "without a norm there are no weights");
  if (!rc && !rotary->norm && ((r.s.heads[0] && !grad_query) || (r.s.heads[1] && !grad_key)))
    rc = fail(MEC_ERR_INVALID, "grad_query and grad_key must be non-null without a norm");
  if (!rc && ((!r.s.heads[0] && grad_query_weight) || (!r.s.heads[1] && grad_key_weight)))
    rc = fail(MEC_ERR_INVALID, "a side without heads has no gradient");
  if (!rc) rc = rotary_groups(r, rotary->norm ? kGradPerCu : kForwardPerCu, &groups);
  const bool weights = grad_query_weight || grad_key_weight;
  if (!rc && weights) rc = check_scratch(workspace, workspace_bytes, (int64_t)groups * 4 * r.s.half * 4);
  if (!rc) rc = check_not_capturing(stream);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (!rotary->norm) {
    // the same turn, backwards
    r.s.sign = -1.f;
    launch_rotary(r, rotary, false, grad_out_query, grad_out_key, grad_query, grad_key, groups, st);
    return check_launch("mec_norm_rotary_backward");
  }
  float* parts = weights ? (float*)workspace : nullptr;
  with_rotary(rotary->dtype, r.vp, rotary->interleaved, [&](auto* t, auto vp, auto il) {
    using T = std::remove_pointer_t<decltype(t)>;
    k_rotary_norm_grad<T, decltype(vp)::value, decltype(il)::value><<<groups, 64 * kRotaryWaves, 0, st>>>(
        r.s, view(query), view(key), view(grad_out_query), view(grad_out_key), (T*)grad_query, (T*)grad_key, parts);
  });
  if (weights) {
    const int d = 2 * r.s.half;
    with_element_type(rotary->weight_dtype, [&](auto* t) {
      using W = std::remove_pointer_t<decltype(t)>;
      k_rotary_dw<W><<<(2 * d + 63) / 64, 64 * kDwWaves, 0, st>>>(parts, groups, d, (W*)grad_query_weight,
                                                                  (W*)grad_key_weight);
    });
  }
  return check_launch("mec_norm_rotary_backward");
}

}  // extern "C"
