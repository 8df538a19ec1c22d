// C-ABI entry points of attention's forward (include/mec.h): argument validation in
// plain host code, then stream-ordered kernel launches.  Nothing here allocates
// device memory or synchronises the host.
#include "mec_attn_fwd.h"
#include "mec_attn_whole.h"
#include "mec_attn_host.h"

using namespace mec;
using namespace mec::attn;

namespace {

// How the forward's work is cut.
struct Plan {
  bool few;        // few rows a key head: the waves of a workgroup share them
  int whole;       // waves of the form for short sequences, 0: not that one
  size_t lds;      // ... and its LDS
  int row_tiles, splits;
  int64_t parts_o, parts_ml;  // bytes
};
constexpr int kWave = 4;

// Waves of k_attn_whole_forward and its LDS, 0 waves where another form is taken: of 16-bit types 48 KB of keys and values
// (three workgroups share a CU), 40 KB beyond 128 keys and up to 256 keys, of fp32 64 KB; and not for few rows of many
// keys, whose loads want more waves.  256 x 12 heads, us, this form and the one that walks over tiles.  bf16, heads of 64: 77
// tokens 27 and 30, 160 (40 KB) 65 and 69, 176 (48 KB) 78 and 72, 225 (64 KB) 109 and 94; of 72: 96 tokens (36 KB) 38 and
// 43, 128 (48 KB) 53 and 54, 160 (60 KB) 122 and 90; of 128: 96 tokens (48 KB) 71 and 72, 128 (64 KB) 95 and 88; of 32: 160
// tokens 33 and 47, 225 (32 KB) 63 and 64, 257 (36 KB) 107 and 94.  fp32, heads of 64: 128 tokens (64 KB) 159 and 191; of
// 32: 160 tokens (40 KB) 159 and 162, 224 (56 KB) 233 and 219, 256 (64 KB) 238 and 246.
int whole_forward(const Problem& a, int dtype, int64_t rows, size_t* lds) {
  const bool f32 = dtype == MEC_DTYPE_F32;
  const int size = f32 ? 4 : 2, steps = a.d <= 32 ? 2 : a.d <= 64 ? 4 : a.d <= 96 ? 6 : 8;
  const int64_t blocks = ceil_div(rows, 32), key_blocks = ceil_div(a.keys, 32);
  const size_t most = f32 ? 64 * 1024 : key_blocks <= 4 ? 48 * 1024 : key_blocks <= 8 ? 40 * 1024 : 0;
  *lds = (size_t)(key_blocks * 2 * 32 * 16 * steps * size);
  // (rows leave through the place of keys and values)
  const bool fits = blocks <= whole_waves(steps, size) && *lds <= most && blocks <= 2 * key_blocks;
  return fits && key_blocks <= 4 * blocks ? (int)blocks : 0;
}

int plan_forward(const Problem& a, int dtype, Plan* out) {
  const int64_t rows = (int64_t)a.queries * a.group;
  Plan p{};
  int cus = 0;
  if (int rc = compute_units(&cus)) return rc;
  // (128 rows a workgroup would leave the device empty: the waves share 32)
  p.few = rows <= 32 || a.pairs * ceil_div(rows, 128) < cus;
  p.row_tiles = (int)ceil_div(rows, p.few ? 32 : 128);
  p.splits = 1;
  p.whole = whole_forward(a, dtype, rows, &p.lds);
  if (p.whole) {
    p.row_tiles = 1;
  } else if (p.few) {
    // two workgroups a CU, and four tiles of 32 keys a wave
    const int64_t want = ceil_div(2 * cus, a.pairs * p.row_tiles), most = ceil_div(a.keys, 32 * kWave * 4);
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
  if (!rc) rc = plan_forward(a, attention->dtype, &p);
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
  if (!rc) rc = plan_forward(a, attention->dtype, &p);
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
    if (p.whole) {
      k_attn_whole_forward<T, KS><<<g.dims, 64 * p.whole, p.lds, st>>>(a, g.items, (T*)out, lse);
    } else if (p.few) {
      k_attn_forward<T, KS, 1, kWave>
          <<<g.dims, 64 * kWave, 0, st>>>(a, g.items, p.row_tiles, p.splits, (T*)out, lse, parts);
      if (p.splits > 1) {
        const int64_t rows = a.pairs * a.queries * a.group, groups = ceil_div(rows, 4);
        const int64_t x = groups < (1 << 20) ? groups : (1 << 20);
        k_attn_join<T><<<dim3((unsigned)x, (unsigned)ceil_div(groups, x)), 256, 0, st>>>(a, rows, p.splits, parts,
                                                                                        (T*)out, lse);
      }
    } else {
      k_attn_forward<T, KS, kWave, 1><<<g.dims, 64 * kWave, 0, st>>>(a, g.items, p.row_tiles, 1, (T*)out, lse, parts);
    }
  });
  return check_launch("mec_attention");
}

}  // extern "C"
