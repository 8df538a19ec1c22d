// C-ABI entry points of the operators over a vocabulary (include/mec.h):
// argument validation in plain host code, then stream-ordered kernel launches.
// Nothing here allocates device memory or synchronises the host.
#include <cmath>

#include "mec_embed.h"
#include "mec_host.h"
#include "mec_vocab.h"

using namespace mec;

namespace {

// (256 threads a row stay below 2^32 work-items)
constexpr int64_t kMaxRows = int64_t(1) << 23;
constexpr int64_t kMaxTokens = int64_t(1) << 23, kMaxEmbedVocab = int64_t(1) << 22, kMaxEmbedDim = int64_t(1) << 16;
constexpr int64_t kMaxStride = int64_t(1) << 40;

// float, bf16 bits or fp16 for dtype
template <class F>
void with_dtype(int dtype, F f) {
  if (dtype == MEC_DTYPE_F32)
    f((float*)nullptr);
  else if (dtype == MEC_DTYPE_BF16)
    f((uint16_t*)nullptr);
  else
    f((_Float16*)nullptr);
}

// f(true_type or false_type): whether an output of this size is stored past the
// last-level cache
template <class F>
void with_past(int64_t bytes, F f) {
  if (bytes > kKeepBytes)
    f(std::true_type{});
  else
    f(std::false_type{});
}

int check_dtype(int dtype) {
  if (dtype != MEC_DTYPE_F32 && dtype != MEC_DTYPE_BF16 && dtype != MEC_DTYPE_F16)
    return fail(MEC_ERR_INVALID, "dtype %d is not MEC_DTYPE_F32, _BF16 or _F16", dtype);
  return MEC_OK;
}

int check_tokens(const void* tokens, int token_bytes) {
  if (tokens == nullptr) return fail(MEC_ERR_INVALID, "tokens must be non-null");
  if (token_bytes != 4 && token_bytes != 8) return fail(MEC_ERR_INVALID, "token_bytes=%d must be 4 or 8", token_bytes);
  return MEC_OK;
}

int check_sizes(int64_t rows, int64_t vocab, int dtype) {
  if (rows < 1) return fail(MEC_ERR_INVALID, "rows=%lld must be >= 1", (long long)rows);
  if (rows > kMaxRows) return fail(MEC_ERR_UNSUPPORTED, "rows=%lld exceeds the maximum 2^23", (long long)rows);
  if (vocab < 1) return fail(MEC_ERR_INVALID, "vocab=%lld must be >= 1", (long long)vocab);
  if (vocab > MEC_MAX_VOCAB) return fail(MEC_ERR_UNSUPPORTED, "vocab=%lld exceeds the maximum 2^19", (long long)vocab);
  return check_dtype(dtype);
}

// A matrix of logits as the callers give it.
struct Logits {
  const void* p;
  int64_t rows, inner, outer_stride, inner_stride, vocab;
  int dtype;
  // (an inner beyond the rows means the same as all of them, and fits the kernels' 32 bits)
  RowMap map() const { return RowMap{inner < rows ? inner : rows, outer_stride, inner_stride}; }
  // every row begins on a 4-byte boundary
  bool aligned() const {
    return dtype == MEC_DTYPE_F32 ||
           (((uintptr_t)p & 3) == 0 && outer_stride % 2 == 0 && (inner == 1 || inner_stride % 2 == 0));
  }
};

int check_logits(const Logits& x) {
  if (int rc = check_sizes(x.rows, x.vocab, x.dtype)) return rc;
  if (x.p == nullptr) return fail(MEC_ERR_INVALID, "logits must be non-null");
  if (x.inner < 1) return fail(MEC_ERR_INVALID, "inner=%lld must be >= 1", (long long)x.inner);
  if (x.outer_stride < 0 || x.inner_stride < 0 || x.outer_stride > kMaxStride || x.inner_stride > kMaxStride)
    return fail(MEC_ERR_INVALID, "row strides %lld, %lld out of range [0, 2^40]", (long long)x.outer_stride,
                (long long)x.inner_stride);
  return MEC_OK;
}

int check_temperature(float t) {
  // (1 / T and log2(e) / T are used: both have to be finite and not 0)
  if (!(t >= 1e-6f && t <= 1e6f)) return fail(MEC_ERR_INVALID, "temperature must be in [1e-6, 1e6]");
  return MEC_OK;
}

int check_top_k(int64_t vocab, int top_k) {
  if (top_k < 0 || top_k > vocab)
    return fail(MEC_ERR_INVALID, "top_k=%d out of range [0, vocab=%lld]", top_k, (long long)vocab);
  if (top_k > MEC_MAX_TOP_K)
    return fail(MEC_ERR_UNSUPPORTED, "top_k=%d exceeds the maximum %d", top_k, MEC_MAX_TOP_K);
  return MEC_OK;
}

int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
  if (need > 0 && workspace == nullptr) return fail(MEC_ERR_INVALID, "workspace must be non-null");
  if (bytes < need)
    return fail(MEC_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)bytes, (long long)need);
  if (((uintptr_t)workspace & 15) != 0) return fail(MEC_ERR_INVALID, "workspace must be 16-byte aligned");
  return MEC_OK;
}

int check_teacher_k(int64_t k) {
  if (k < 1) return fail(MEC_ERR_INVALID, "k=%lld must be >= 1", (long long)k);
  if (k > MEC_MAX_TEACHER_K)
    return fail(MEC_ERR_UNSUPPORTED, "k=%lld exceeds the maximum %d", (long long)k, MEC_MAX_TEACHER_K);
  return MEC_OK;
}

int check_teacher(const void* tokens, int token_bytes, const void* logits, int dtype, int64_t k) {
  if (int rc = check_tokens(tokens, token_bytes)) return rc;
  if (logits == nullptr) return fail(MEC_ERR_INVALID, "teacher_logits must be non-null");
  if (int rc = check_teacher_k(k)) return rc;
  return check_dtype(dtype);
}

int check_loss(float temperature, float weight, int reduction) {
  if (int rc = check_temperature(temperature)) return rc;
  if (!std::isfinite(weight)) return fail(MEC_ERR_INVALID, "weight must be finite");
  if (reduction != MEC_REDUCE_NONE && reduction != MEC_REDUCE_SUM && reduction != MEC_REDUCE_MEAN)
    return fail(MEC_ERR_INVALID, "unknown reduction %d", reduction);
  return MEC_OK;
}

int check_embedding(const void* tokens, int token_bytes, int64_t n, int64_t vocab, int64_t d, int dtype, float scale) {
  if (int rc = check_tokens(tokens, token_bytes)) return rc;
  if (n < 1 || vocab < 1 || d < 1)
    return fail(MEC_ERR_INVALID, "n=%lld, vocab=%lld, d=%lld must be >= 1", (long long)n, (long long)vocab,
                (long long)d);
  if (n > kMaxTokens || vocab > kMaxEmbedVocab || d > kMaxEmbedDim)
    return fail(MEC_ERR_UNSUPPORTED, "n=%lld, vocab=%lld, d=%lld exceed the maxima 2^23, 2^22, 2^16", (long long)n,
                (long long)vocab, (long long)d);
  if (!std::isfinite(scale)) return fail(MEC_ERR_INVALID, "scale must be finite");
  return check_dtype(dtype);
}

int64_t round16(int64_t b) { return (b + 15) & ~int64_t(15); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How token scores cut a row.
struct Cut {
  int segments, len;
  uint32_t rows_x(int64_t rows) const {
    const int64_t most = (int64_t(1) << 23) / segments;
    return (uint32_t)(rows < most ? rows : most);
  }
  SegmentGrid grid(int64_t rows) const { return SegmentGrid{segments, len, rows_x(rows)}; }
  dim3 dims(int64_t rows) const {
    return dim3(rows_x(rows) * segments, (unsigned)((rows + rows_x(rows) - 1) / rows_x(rows)));
  }
};
constexpr int64_t kManyRows = 1024;  // a workgroup each fills the device
Cut cut_rows(int64_t rows, int64_t vocab, int dtype, bool aligned) {
  const int64_t vec = dtype == MEC_DTYPE_F32 ? 4 : 8, chunk = kRowThreads * vec;  // a vector per thread
  if (!aligned) ++vocab;  // counted from the boundary before the row
  int64_t s = ceil_div(vocab, chunk * kSegChunks);
  // few rows: more, shorter segments, so that there are workgroups for every CU
  const int64_t want = ceil_div(kManyRows, rows);
  if (s < want) s = want;
  if (s > ceil_div(vocab, chunk)) s = ceil_div(vocab, chunk);
  if (s > kMaxSegments) s = kMaxSegments;
  const int64_t len = ceil_div(ceil_div(vocab, s), chunk) * chunk;
  return Cut{(int)ceil_div(vocab, len), (int)len};
}
// most segments of a row, wherever its rows begin
int64_t most_segments(int64_t rows, int64_t vocab, int dtype) {
  const int a = cut_rows(rows, vocab, dtype, true).segments, b = cut_rows(rows, vocab, dtype, false).segments;
  return a > b ? a : b;
}
int64_t scores_parts_bytes(int64_t rows, const Cut& c) { return c.segments > 1 ? rows * c.segments * 16 : 0; }
int64_t scores_workspace(int64_t rows, int64_t vocab, int top_k, int dtype) {
  const int64_t s = most_segments(rows, vocab, dtype);
  return s > 1 ? rows * s * 16 + round16(rows * s * top_k * 8) : 0;
}

// The workgroup that makes a row's loss and gradient: the fewest threads that hold
// it in registers, else several segments.
struct RowShape {
  int threads, segments, len;
};
RowShape row_shape(int64_t vocab, int dtype, bool aligned) {
  const int64_t vec = dtype == MEC_DTYPE_F32 ? 4 : 8;
  for (int threads = 256; threads <= 1024; threads *= 2)
    if (vocab + (aligned ? 0 : 1) <= vec * kSegChunks * threads) return RowShape{threads, 1, (int)vocab};
  // Two workgroups of 512 threads on a CU read and write at the same time, one of
  // 1024 holds twice as much of a row.  512 / 1024 threads, with rows for every CU
  // (fewer were not compared), bf16: 8192 x 70001 512 / 697 us, 4096 x 128256 442 /
  // 508, 4096 x 200000 705 / 729, 4096 x 212000 794 / 760, 2048 x 250002 530 / 483;
  // fp32 (half the arithmetic a byte): 4096 x 36000 239 / 297, 4096 x 49408 342 / 368,
  // 2048 x 70000 262 / 258, 2048 x 100003 403 / 378.
  const int threads = vocab <= (dtype == MEC_DTYPE_F32 ? 65536 : 204800) ? 512 : 1024;
  // (the first segment may begin off a boundary, and end up to a vector later for it)
  const int64_t len = vec * kSegChunks * threads - (aligned ? 0 : vec);
  return RowShape{threads, (int)ceil_div(vocab, len), (int)len};
}

// Workspace of mec_distill_forward, in bytes from its start.
struct DistillWorkspace {
  int64_t some, counts, row_loss, parts, total;
};
DistillWorkspace distill_workspace(int64_t rows, int64_t vocab, int dtype, bool with_grad) {
  DistillWorkspace w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += round16(bytes);
    return p;
  };
  w.some = take(rows * 4);
  w.counts = take(kTeacherGroups * 4);
  w.row_loss = take(rows * 4);
  w.parts = take(with_grad ? 0 : rows * most_segments(rows, vocab, dtype) * 8);
  w.total = at;
  return w;
}

// Workspace of mec_embedding_backward, in bytes from its start.
struct EmbedWorkspace {
  int64_t even, odd, keys, positions, bounds, counts, pieces, blocks, total;
};
EmbedWorkspace embed_workspace(int64_t n, int64_t vocab, int64_t d) {
  EmbedWorkspace w{};
  if (n <= kFew) return w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += round16(bytes);
    return p;
  };
  w.even = take(n * 8);
  w.odd = take(n * 8);
  w.keys = take(n * 4);
  w.positions = take(n * 4);
  w.bounds = take(vocab * 8);
  w.counts = take((ceil_div(n, (int64_t)kSortThreads * kSortItems) + kSortTiles + 1) * kSortBins * 4);
  w.pieces = take(n / kPiece * d * 4);
  w.blocks = take(n / kBlock * d * 4);
  w.total = at;
  return w;
}

// Sorted tokens and their positions into the workspace.
Runs sort_tokens(const void* tokens, int token_bytes, int64_t n, int64_t vocab, int64_t padding,
                 const EmbedWorkspace& w, char* ws, hipStream_t st) {
  int key_bits = 1;
  while ((vocab >> key_bits) != 0) ++key_bits;
  const int passes = (key_bits + 8) / 9, bits = (key_bits + passes - 1) / passes;
  // pairs per lane: as few as keep the tiles within kSortTiles
  const int64_t per_lane = ceil_div(n, n <= kSortOne ? kSortOneThreads : (int64_t)kSortThreads * kSortTiles);
  SortShape s{n, (int)(per_lane < kSortItems ? per_lane : kSortItems), 1, (int)vocab, padding};
  const Tokens tok{tokens, token_bytes == 8};
  uint2 *even = (uint2*)(ws + w.even), *odd = (uint2*)(ws + w.odd);
  const SortOut last{nullptr, (int*)(ws + w.keys), (int*)(ws + w.positions)};
  int2* bounds = (int2*)(ws + w.bounds);
  if (n <= kSortOne) {
    const int64_t clears = ceil_div(vocab, 4 * kSortOneThreads);
    const unsigned groups = 1 + (unsigned)(clears < 256 ? clears : 256);
    k_sort_one<<<groups, kSortOneThreads, 0, st>>>(tok, s, passes, bits, even, odd, last, bounds);
  } else {
    s.tiles = (int)ceil_div(n, (int64_t)kSortThreads * s.items);
    int* counts = (int*)(ws + w.counts);
    for (int pass = 0; pass < passes; ++pass) {
      const SortSource src{tok, pass == 0 ? nullptr : pass & 1 ? even : odd};
      const SortOut out = pass == passes - 1 ? last : SortOut{pass & 1 ? odd : even, nullptr, nullptr};
      k_sort_count<<<s.tiles, kSortThreads, 0, st>>>(src, s, pass * bits, bits, counts, pass == 0 ? bounds : nullptr);
      if (s.tiles > kSortTiles) k_sort_prefix<<<kSortBins / 64, kSortThreads, 0, st>>>(counts, s.tiles);
      k_sort_scatter<<<s.tiles, kSortThreads, 0, st>>>(src, s, pass * bits, bits, counts, out);
    }
  }
  return Runs{last.keys, last.positions, n, (int)vocab, bounds};
}

}  // namespace

extern "C" {

int64_t mec_token_scores_workspace_bytes(int64_t rows, int64_t vocab, int top_k, int dtype) {
  g_err.clear();
  int rc = check_sizes(rows, vocab, dtype);
  if (!rc) rc = check_top_k(vocab, top_k);
  return rc ? rc : scores_workspace(rows, vocab, top_k, dtype);
}

int mec_token_scores(const void* logits, int64_t rows, int64_t inner, int64_t outer_stride, int64_t inner_stride,
                     int64_t vocab, int dtype, const void* tokens, int token_bytes, int64_t ignore_index,
                     float temperature, int top_k, float* log_probs, float* entropy, int64_t* top_tokens,
                     float* top_log_probs, float* state, void* workspace, int64_t workspace_bytes, void* stream) {
  g_err.clear();
  const Logits x{logits, rows, inner, outer_stride, inner_stride, vocab, dtype};
  int rc = check_logits(x);
  if (!rc) rc = check_tokens(tokens, token_bytes);
  if (!rc) rc = check_temperature(temperature);
  if (!rc) rc = check_top_k(vocab, top_k);
  if (!rc && (!log_probs || !entropy || (top_k > 0 && (!top_tokens || !top_log_probs))))
    rc = fail(MEC_ERR_INVALID, "outputs must be non-null");
  if (!rc) rc = check_workspace(workspace, workspace_bytes, scores_workspace(rows, vocab, top_k, dtype));
  if (!rc) rc = check_not_capturing(stream);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const T* p = (const T*)logits;
    const Tokens tok{tokens, token_bytes == 8};
    const Cut cut = cut_rows(rows, vocab, dtype, x.aligned());
    float4* parts = (float4*)workspace;
    uint64_t* part_top = (uint64_t*)((char*)workspace + scores_parts_bytes(rows, cut));
    const ScoresOut out{log_probs, entropy, top_tokens, top_log_probs, state};
    const dim3 grid = cut.dims(rows);
    const float inv_t = 1.f / temperature;
    if (top_k > 0)
      k_scores<T, true><<<grid, kRowThreads, 0, st>>>(p, x.map(), (int)vocab, tok, ignore_index, inv_t, top_k, out,
                                                      rows, cut.grid(rows), parts, part_top);
    else
      k_scores<T, false><<<grid, kRowThreads, 0, st>>>(p, x.map(), (int)vocab, tok, ignore_index, inv_t, 0, out, rows,
                                                       cut.grid(rows), parts, part_top);
    if (cut.segments > 1)
      k_scores_join<T><<<(unsigned)rows, kJoinThreads, (size_t)cut.segments * top_k * 8, st>>>(
          p, x.map(), (int)vocab, tok, ignore_index, inv_t, top_k, out, rows, cut.segments, parts, part_top);
  });
  return check_launch("mec_token_scores");
}

int mec_token_scores_backward(const void* logits, int64_t rows, int64_t inner, int64_t outer_stride,
                              int64_t inner_stride, int64_t vocab, int dtype, const void* tokens, int token_bytes,
                              int64_t ignore_index, float temperature, const float* state, const float* entropy,
                              const float* grad_log_probs, const float* grad_entropy, void* grad_logits,
                              void* stream) {
  g_err.clear();
  const Logits x{logits, rows, inner, outer_stride, inner_stride, vocab, dtype};
  int rc = check_logits(x);
  if (!rc) rc = check_tokens(tokens, token_bytes);
  if (!rc) rc = check_temperature(temperature);
  if (!rc && (!state || !entropy || !grad_logits))
    rc = fail(MEC_ERR_INVALID, "state, entropy and grad_logits must be non-null");
  if (!rc) rc = check_not_capturing(stream);
  if (rc) return rc;
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const Cut cut = cut_rows(kManyRows, vocab, dtype, x.aligned());
    with_past(rows * vocab * sizeof(T), [&](auto past) {
      k_scores_grad<T, decltype(past)::value><<<cut.dims(rows), kRowThreads, 0, (hipStream_t)stream>>>(
          (const T*)logits, x.map(), (int)vocab, Tokens{tokens, token_bytes == 8}, ignore_index, 1.f / temperature,
          state, entropy, grad_log_probs, grad_entropy, (T*)grad_logits, rows, cut.grid(rows));
    });
  });
  return check_launch("mec_token_scores_backward");
}

int64_t mec_distill_workspace_bytes(int64_t rows, int64_t vocab, int64_t k, int dtype, int with_grad) {
  g_err.clear();
  int rc = check_sizes(rows, vocab, dtype);
  if (!rc) rc = check_teacher_k(k);
  return rc ? rc : distill_workspace(rows, vocab, dtype, with_grad != 0).total;
}

int mec_distill_forward(const void* logits, int64_t rows, int64_t inner, int64_t outer_stride, int64_t inner_stride,
                        int64_t vocab, int dtype, const void* teacher_tokens, int token_bytes,
                        const void* teacher_logits, int teacher_dtype, int64_t k, float temperature, float weight,
                        int reduction, float* loss, float* state, void* grad_logits, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  g_err.clear();
  const Logits x{logits, rows, inner, outer_stride, inner_stride, vocab, dtype};
  int rc = check_logits(x);
  if (!rc) rc = check_teacher(teacher_tokens, token_bytes, teacher_logits, teacher_dtype, k);
  if (!rc) rc = check_loss(temperature, weight, reduction);
  if (!rc && (!loss || !state)) rc = fail(MEC_ERR_INVALID, "loss and state must be non-null");
  if (!rc && grad_logits && reduction == MEC_REDUCE_NONE)
    rc = fail(MEC_ERR_INVALID, "grad_logits needs MEC_REDUCE_SUM or MEC_REDUCE_MEAN");
  const DistillWorkspace w = rc ? DistillWorkspace{} : distill_workspace(rows, vocab, dtype, grad_logits != nullptr);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, w.total);
  if (!rc) rc = check_not_capturing(stream);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  const Teacher teacher{{teacher_tokens, token_bytes == 8}, teacher_logits, teacher_dtype, (int)k};
  char* ws = (char*)workspace;
  const int64_t each = ceil_div(ceil_div(rows, kTeacherGroups), kTeacherRows) * kTeacherRows;
  const TeacherRows have{(int*)(ws + w.some), (int*)(ws + w.counts), (int)ceil_div(rows, each), (int)each};
  k_teacher_rows<<<have.groups, kTeacherThreads, 0, st>>>(teacher, rows, have);
  float* row_loss = reduction == MEC_REDUCE_NONE ? loss : (float*)(ws + w.row_loss);
  const DistillState ds{state, state + rows};
  const float inv_t = 1.f / temperature;
  const int mean = reduction == MEC_REDUCE_MEAN;
  const size_t lds = (size_t)k * 12;
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const T* p = (const T*)logits;
    const int n = (int)vocab;
    if (grad_logits) {
      const RowShape shape = row_shape(vocab, dtype, x.aligned());
      auto run = [&](auto threads, auto one) {
        constexpr int THREADS = decltype(threads)::value;
        with_past(rows * vocab * sizeof(T), [&](auto past) {
          k_distill_row<T, THREADS, decltype(one)::value, decltype(past)::value><<<(unsigned)rows, THREADS, lds, st>>>(
              p, x.map(), n, teacher, inv_t, weight, have, mean, row_loss, ds, (T*)grad_logits, shape.segments,
              shape.len);
        });
      };
      const bool one = shape.segments == 1;
      if (shape.threads == 256)
        run(std::integral_constant<int, 256>{}, std::true_type{});
      else if (shape.threads == 512 && one)
        run(std::integral_constant<int, 512>{}, std::true_type{});
      else if (shape.threads == 512)
        run(std::integral_constant<int, 512>{}, std::false_type{});
      else if (one)
        run(std::integral_constant<int, 1024>{}, std::true_type{});
      else
        run(std::integral_constant<int, 1024>{}, std::false_type{});
      return;
    }
    const Cut cut = cut_rows(rows, vocab, dtype, x.aligned());
    float2* parts = (float2*)(ws + w.parts);
    k_distill_sums<T><<<cut.dims(rows), kRowThreads, 0, st>>>(p, x.map(), n, inv_t, have.some, rows, cut.grid(rows),
                                                              parts);
    k_distill_join<T><<<(unsigned)rows, 64, lds, st>>>(p, x.map(), n, teacher, inv_t, weight, have.some, parts,
                                                       cut.segments, row_loss, ds);
  });
  if (reduction != MEC_REDUCE_NONE)
    k_loss_sum<<<1, kSumThreads, 0, st>>>(row_loss, rows, have, mean, (int*)(state + 2 * rows), loss);
  return check_launch("mec_distill_forward");
}

int mec_distill_backward(const void* logits, int64_t rows, int64_t inner, int64_t outer_stride, int64_t inner_stride,
                         int64_t vocab, int dtype, const void* teacher_tokens, int token_bytes,
                         const void* teacher_logits, int teacher_dtype, int64_t k, float temperature, float weight,
                         int reduction, const float* state, const float* grad_output, int made, void* grad_logits,
                         void* stream) {
  g_err.clear();
  const Logits x{logits, rows, inner, outer_stride, inner_stride, vocab, dtype};
  int rc = check_logits(x);
  if (!rc) rc = check_teacher(teacher_tokens, token_bytes, teacher_logits, teacher_dtype, k);
  if (!rc) rc = check_loss(temperature, weight, reduction);
  if (!rc && (!state || !grad_output || !grad_logits))
    rc = fail(MEC_ERR_INVALID, "state, grad_output and grad_logits must be non-null");
  if (!rc && made && reduction == MEC_REDUCE_NONE)
    rc = fail(MEC_ERR_INVALID, "made needs MEC_REDUCE_SUM or MEC_REDUCE_MEAN");
  if (!rc) rc = check_not_capturing(stream);
  if (rc) return rc;
  const Teacher teacher{{teacher_tokens, token_bytes == 8}, teacher_logits, teacher_dtype, (int)k};
  const int* count = reduction == MEC_REDUCE_MEAN ? (const int*)(state + 2 * rows) : nullptr;
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const Cut cut = cut_rows(kManyRows, vocab, dtype, x.aligned());
    const int64_t items = rows * cut.segments;
    // (made: few workgroups are enough to find that grad_output is 1)
    const int64_t most = made ? 2048 : int64_t(1) << 22;
    with_past(rows * vocab * sizeof(T), [&](auto past) {
      k_distill_grad<T, decltype(past)::value>
          <<<(unsigned)(items < most ? items : most), kRowThreads, (size_t)k * 12, (hipStream_t)stream>>>(
              (const T*)logits, x.map(), (int)vocab, teacher, 1.f / temperature, weight, count,
              DistillState{const_cast<float*>(state), const_cast<float*>(state) + rows}, grad_output,
              reduction == MEC_REDUCE_NONE, made, (T*)grad_logits, rows, cut.len, cut.segments);
    });
  });
  return check_launch("mec_distill_backward");
}

int mec_embedding(const void* tokens, int token_bytes, int64_t n, const void* weight, int64_t ldw, int64_t vocab,
                  int64_t d, int dtype, float scale, void* out, void* stream) {
  g_err.clear();
  int rc = check_embedding(tokens, token_bytes, n, vocab, d, dtype, scale);
  if (!rc && (!weight || !out)) rc = fail(MEC_ERR_INVALID, "weight and out must be non-null");
  if (!rc && (ldw < d || ldw > kMaxStride))
    rc = fail(MEC_ERR_INVALID, "row stride ldw=%lld must be in [d=%lld, 2^40]", (long long)ldw, (long long)d);
  if (!rc) rc = check_not_capturing(stream);
  if (rc) return rc;
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    int lg = 0;  // lanes for a row: up to a wave, one vector each
    while (lg < 6 && (int64_t)Vec<T>::N << lg < d) ++lg;
    const int64_t per_group = (kEmbedThreads >> lg) * kEmbedTokens;
    with_past(n * d * sizeof(T), [&](auto past) {
      k_embed<T, decltype(past)::value>
          <<<(unsigned)ceil_div(n, per_group), kEmbedThreads, 0, (hipStream_t)stream>>>(
              Tokens{tokens, token_bytes == 8}, n, (const T*)weight, ldw, vocab, (int)d, lg, scale, (T*)out);
    });
  });
  return check_launch("mec_embedding");
}

int64_t mec_embedding_workspace_bytes(int64_t n, int64_t vocab, int64_t d, int dtype) {
  g_err.clear();
  int rc = check_embedding((const void*)1, 8, n, vocab, d, dtype, 1.f);
  return rc ? rc : embed_workspace(n, vocab, d).total;
}

int mec_embedding_backward(const void* tokens, int token_bytes, int64_t n, const void* grad_out, int64_t ldg,
                           int64_t vocab, int64_t d, int dtype, float scale, int64_t padding_idx, void* grad_weight,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  g_err.clear();
  int rc = check_embedding(tokens, token_bytes, n, vocab, d, dtype, scale);
  if (!rc && (!grad_out || !grad_weight)) rc = fail(MEC_ERR_INVALID, "grad_out and grad_weight must be non-null");
  if (!rc && (ldg < d || ldg > kMaxStride))
    rc = fail(MEC_ERR_INVALID, "row stride ldg=%lld must be in [d=%lld, 2^40]", (long long)ldg, (long long)d);
  if (!rc && (padding_idx < -1 || padding_idx >= vocab))
    rc = fail(MEC_ERR_INVALID, "padding_idx=%lld out of range [-1, vocab=%lld)", (long long)padding_idx,
              (long long)vocab);
  const EmbedWorkspace w = rc ? EmbedWorkspace{} : embed_workspace(n, vocab, d);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, w.total);
  if (!rc) rc = check_not_capturing(stream);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  float *pieces = (float*)(ws + w.pieces), *blocks = (float*)(ws + w.blocks);
  const FewTokens few{{tokens, token_bytes == 8}, padding_idx};
  const Runs runs = n <= kFew ? Runs{nullptr, nullptr, n, (int)vocab, nullptr}
                              : sort_tokens(tokens, token_bytes, n, vocab, padding_idx, w, ws, st);
  with_dtype(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int N = Vec<T>::N;
    if (runs.bounds) {
      const dim3 grid((unsigned)ceil_div(n, kBlock), (unsigned)ceil_div(d, 64 * N));
      k_embed_pieces<T><<<grid, kBlockPieces * 64, 0, st>>>(runs, (const T*)grad_out, ldg, (int)d, pieces, blocks);
    }
    const unsigned groups = (unsigned)ceil_div(vocab, kDwRows);
    auto rows = [&](auto nc) {
      constexpr int NC = decltype(nc)::value;
      with_past(vocab * d * sizeof(T), [&](auto past) {
        k_embed_rows<T, NC, decltype(past)::value><<<dim3(groups, (unsigned)ceil_div(d, NC * 64 * N)), 256, 0, st>>>(
            runs, few, (const T*)grad_out, ldg, (int)d, scale, pieces, blocks, (T*)grad_weight);
      });
    };
    // (1024 columns by a wave: more of them in 16 bits take too many registers)
    if (d <= 64 * N) return rows(std::integral_constant<int, 1>{});
    if constexpr (sizeof(T) == 4)
      if (d > 128 * N) return rows(std::integral_constant<int, 4>{});
    rows(std::integral_constant<int, 2>{});
  });
  return check_launch("mec_embedding_backward");
}

}  // extern "C"
