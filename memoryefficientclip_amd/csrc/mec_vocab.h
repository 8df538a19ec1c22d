// Kernels over rows of logits of a vocabulary: log probabilities of given
// tokens with entropy and top alternatives, and distillation from a teacher's
// top logits, each with its gradient.
//
// A row x_0 .. x_{V-1} at temperature T, c = log2(e) / T:
//   m = max x,  t_v = (x_v - m) c,  S = sum 2^t_v,  U = sum 2^t_v t_v
//   log p_v = ln2 t_v - ln S,  entropy = ln S - ln2 U / S
// A row of nothing but -inf has S = 0: p = 0, log p = -inf, entropy 0.  A NaN or
// +inf makes S NaN, and with it all that is formed from the row.
#pragma once
#include "mec_common.h"

namespace mec {

constexpr float kLn2 = 0.69314718055994531f;

// Row r starts at (r / inner) * outer_stride + (r % inner) * inner_stride
// elements (64 bits: a matrix of logits passes 2^32 elements).
struct RowMap {
  int64_t inner, outer_stride, inner_stride;
  __device__ __forceinline__ int64_t operator()(int64_t r) const {
    return inner == 1 ? r * outer_stride : (r / inner) * outer_stride + (r % inner) * inner_stride;
  }
};

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float value(_Float16 v) { return (float)v; }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = f32_to_bf16(v); }
__device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }

// Token i of an int64 or int32 array.
struct Tokens {
  const void* p;
  int wide;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
  }
};

// Order of the alternatives as a number: larger values first, NaN before
// everything, -0 like +0; among equal ones the lower index first.
__device__ __forceinline__ uint32_t order_bits(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(float v, int index) {
  return ((uint64_t)order_bits(v) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u >> 31) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)~(uint32_t)key; }

// (x - m) / T where the difference itself may pass fp32's range
__device__ __forceinline__ float scaled_difference(float x, float m, float inv_t) {
  return (0.5f * x - 0.5f * m) * (2.f * inv_t);
}

constexpr int kRowThreads = 256;

template <class V, class Op>
__device__ __forceinline__ V block_reduce(V v, V* lds, Op op) {
  for (int m = 32; m >= 1; m >>= 1) v = op(v, (V)__shfl_xor(v, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < kRowThreads / 64; ++w) v = op(v, lds[w]);
  return v;
}

struct RowSums {
  float m, s, u;
};

// m, S and U of a row, in every thread.
template <class T, bool U>
__device__ __forceinline__ RowSums row_sums(const T* x, int n, float c, float* lds) {
  float m = -INFINITY;
  for (int v = threadIdx.x; v < n; v += kRowThreads) m = fmaxf(m, value(x[v]));
  m = block_reduce(m, lds, [](float a, float b) { return fmaxf(a, b); });
  const float ref = m == -INFINITY ? 0.f : m;
  float s = 0.f, u = 0.f;
  for (int v = threadIdx.x; v < n; v += kRowThreads) {
    const float t = (value(x[v]) - ref) * c;
    const float e = fast_exp2(t);
    s += e;
    // (2^t is 0 below -200, where t may be -inf)
    if (U) u += e * fmaxf(t, -200.f);
  }
  s = block_reduce(s, lds, [](float a, float b) { return a + b; });
  if (U) u = block_reduce(u, lds, [](float a, float b) { return a + b; });
  return {ref, s, u};
}

// One workgroup per row.
template <class T>
__global__ __launch_bounds__(kRowThreads) void k_token_scores(const T* logits, RowMap map, int n, Tokens tokens,
                                                              int64_t ignore, float inv_t, int k, float* log_probs,
                                                              float* entropy, int64_t* top_tokens,
                                                              float* top_log_probs, float* stats, int64_t rows) {
  __shared__ float lds[kRowThreads / 64];
  __shared__ uint64_t lds64[kRowThreads / 64];
  const int64_t r = blockIdx.x;
  const int64_t tok = tokens[r];
  const int tid = threadIdx.x;
  if (tok == ignore) {
    if (tid == 0) log_probs[r] = 0.f, entropy[r] = 0.f, stats[r] = 0.f, stats[rows + r] = 0.f;
    for (int j = tid; j < k; j += kRowThreads) top_tokens[r * k + j] = -1, top_log_probs[r * k + j] = 0.f;
    return;
  }
  const T* x = logits + map(r);
  const RowSums a = row_sums<T, true>(x, n, inv_t / kLn2, lds);
  const float ls = logf(a.s);
  auto log_prob = [&](float v) { return a.s == 0.f ? -INFINITY : scaled_difference(v, a.m, inv_t) - ls; };
  if (tid == 0) {
    log_probs[r] = tok >= 0 && tok < n ? log_prob(value(x[tok])) : NAN;
    entropy[r] = a.s == 0.f ? 0.f : ls - kLn2 * (a.u / a.s);
    stats[r] = a.m;
    stats[rows + r] = a.s;
  }
  uint64_t last = 0;
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    for (int v = tid; v < n; v += kRowThreads) {
      const uint64_t q = order_key(value(x[v]), v);
      if ((j == 0 || q < last) && q > best) best = q;
    }
    best = block_reduce(best, lds64, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
    last = best;
    if (tid == 0) {
      top_tokens[r * k + j] = key_index(best);
      top_log_probs[r * k + j] = log_prob(value(x[key_index(best)]));
    }
  }
}

// dx_v = (1/T) (g_l (1[v = tok] - p_v) - g_h p_v (log p_v + entropy))
template <class T>
__global__ __launch_bounds__(kRowThreads) void k_token_scores_grad(const T* logits, RowMap map, int n, Tokens tokens,
                                                                   int64_t ignore, float inv_t, const float* stats,
                                                                   const float* entropy, const float* g_log_probs,
                                                                   const float* g_entropy, T* dx, int64_t rows) {
  const int64_t r = blockIdx.x;
  const int64_t tok = tokens[r];
  const T* x = logits + map(r);
  T* y = dx + r * n;
  const float m = stats[r], s = stats[rows + r], h = entropy[r];
  const bool none = tok == ignore || s == 0.f, bad = tok < 0 || tok >= n;
  const float gl = g_log_probs ? g_log_probs[r] : 0.f, gh = g_entropy ? g_entropy[r] : 0.f;
  const float ls = logf(s), inv_s = 1.f / s;
  for (int v = threadIdx.x; v < n; v += kRowThreads) {
    float d = 0.f;
    if (!none) {
      const float z = fmaxf((value(x[v]) - m) * inv_t, -200.f);
      const float p = fast_exp2(z * (1.f / kLn2)) * inv_s;
      d = inv_t * ((v == tok ? gl : 0.f) - p * (gl + gh * (z - ls + h)));
      if (value(x[v]) != value(x[v]) || bad) d = NAN;
    }
    put(y + v, d);
  }
}

// ---- distillation from a teacher's top logits ----
//
// q = softmax over the row's teacher entries of teacher / T (an entry with a
// token < 0 has none), p = softmax over the vocabulary of x / T:
//   loss_r = scale T^2 sum_j q_j (log q_j - log p_tok_j)
//   dx_v = g scale T (p_v - sum_{j: tok_j = v} q_j)
// A row whose teacher has nothing above -inf has loss 0 and gradient 0; a token
// past the vocabulary makes both NaN.

constexpr int kMaxTeacher = 1024;  // entries per row

struct Teacher {
  Tokens tokens;
  const void* logits;
  int dtype;  // MEC_DTYPE_F32, _BF16, _F16
  int k;
  __device__ __forceinline__ float logit(int64_t i) const {
    return dtype == 0   ? ((const float*)logits)[i]
           : dtype == 1 ? value(((const uint16_t*)logits)[i])
                        : value(((const _Float16*)logits)[i]);
  }
};

// One row's teacher in shared memory.
struct TeacherRow {
  float q[kMaxTeacher], log_q[kMaxTeacher];
  int tok[kMaxTeacher];
  int some, bad;
};

// By the first wave of the workgroup; the caller synchronizes.
__device__ __forceinline__ void load_teacher(const Teacher& t, int64_t r, int n, float inv_t, TeacherRow& row) {
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  const float c = inv_t / kLn2;
  float m = -INFINITY;
  bool bad = false;
  for (int j = lane; j < t.k; j += 64) {
    const int64_t tok = t.tokens[r * t.k + j];
    const float z = tok < 0 ? -INFINITY : t.logit(r * t.k + j);
    bad |= tok >= n;
    row.tok[j] = tok < 0 || tok >= n ? -1 : (int)tok;
    row.log_q[j] = z;
    m = fmaxf(m, z);
  }
  for (int i = 32; i >= 1; i >>= 1) m = fmaxf(m, __shfl_xor(m, i, 64));
  if (m == -INFINITY) m = 0.f;
  float s = 0.f;
  for (int j = lane; j < t.k; j += 64) s += fast_exp2((row.log_q[j] - m) * c);
  s = wave_sum(s);
  const float ls = logf(s);
  for (int j = lane; j < t.k; j += 64) {
    const float z = row.log_q[j] - m;
    row.q[j] = s == 0.f ? 0.f : fast_exp2(z * c) / s;
    row.log_q[j] = z * inv_t - ls;
  }
  bad = __any(bad);
  if (lane == 0) row.some = !(s == 0.f), row.bad = bad;
}

// Rows that have a teacher: one wave per row.
__global__ __launch_bounds__(64) void k_teacher_count(Teacher t, int* count) {
  const int64_t r = blockIdx.x;
  bool some = false;
  for (int j = threadIdx.x; j < t.k; j += 64)
    some |= t.tokens[r * t.k + j] >= 0 && t.logit(r * t.k + j) != -INFINITY;
  if (__any(some) && threadIdx.x == 0) atomicAdd(count, 1);
}

// dx of a row: g (p_v - q at the teacher's tokens).
template <class T>
__device__ __forceinline__ void distill_row_grad(const T* x, T* y, int n, float inv_t, float m, float s, float g,
                                                 const TeacherRow& row, int k) {
  const float c = inv_t / kLn2;
  const bool zero = !row.some || s == 0.f;
  const float gs = row.bad ? NAN : g / s;
  for (int v = threadIdx.x; v < n; v += kRowThreads)
    put(y + v, zero ? 0.f : fast_exp2((value(x[v]) - m) * c) * gs);
  if (zero || row.bad) return;
  __syncthreads();
  // the teacher's tokens once more, each by one thread with all its entries
  for (int j = threadIdx.x; j < k; j += kRowThreads) {
    const int v = row.tok[j];
    if (v < 0) continue;
    float q = 0.f;
    for (int i = 0; i < k; ++i) q += row.tok[i] == v ? row.q[i] : 0.f;
    put(y + v, g * (fast_exp2((value(x[v]) - m) * c) / s - q));
  }
}

// loss, and with dx its gradient for grad_output 1.  count: rows that have a
// teacher (mean), null for 1.
template <class T>
__global__ __launch_bounds__(kRowThreads) void k_distill(const T* logits, RowMap map, int n, Teacher teacher,
                                                         float inv_t, float scale, const int* count, float* row_loss,
                                                         float* stats, T* dx, int64_t rows) {
  __shared__ float lds[kRowThreads / 64];
  __shared__ TeacherRow row;
  const int64_t r = blockIdx.x;
  load_teacher(teacher, r, n, inv_t, row);
  __syncthreads();
  const T* x = logits + map(r);
  RowSums a{0.f, 1.f, 0.f};
  if (row.some) a = row_sums<T, false>(x, n, inv_t / kLn2, lds);
  const float ls = logf(a.s);
  float loss = 0.f;
  for (int j = threadIdx.x; j < teacher.k; j += kRowThreads)
    if (!(row.q[j] == 0.f) && row.tok[j] >= 0)
      loss += row.q[j] * (row.log_q[j] - (a.s == 0.f ? -INFINITY : scaled_difference(value(x[row.tok[j]]), a.m, inv_t) - ls));
  loss = block_reduce(loss, lds, [](float p, float q) { return p + q; });
  if (threadIdx.x == 0) {
    row_loss[r] = row.bad ? NAN : loss * (scale / (inv_t * inv_t));
    stats[r] = a.m;
    stats[rows + r] = a.s;
  }
  if (!dx) return;
  const float rows_in = count ? fmaxf((float)*count, 1.f) : 1.f;
  distill_row_grad(x, dx + r * n, n, inv_t, a.m, a.s, scale / (inv_t * rows_in), row, teacher.k);
}

// dx for a given grad_output (one number, or one for each row).  With
// made = 1 the forward has left the gradient for grad_output 1 in dx.
template <class T>
__global__ __launch_bounds__(kRowThreads) void k_distill_grad(const T* logits, RowMap map, int n, Teacher teacher,
                                                              float inv_t, float scale, const int* count,
                                                              const float* stats, const float* grad_output,
                                                              int per_row, int made, T* dx, int64_t rows) {
  __shared__ TeacherRow row;
  const int64_t r = blockIdx.x;
  const float go = grad_output[per_row ? r : 0];
  if (made && go == 1.f) return;
  load_teacher(teacher, r, n, inv_t, row);
  __syncthreads();
  const float rows_in = count ? fmaxf((float)*count, 1.f) : 1.f;
  distill_row_grad(logits + map(r), dx + r * n, n, inv_t, stats[r], stats[rows + r], go * scale / (inv_t * rows_in),
                   row, teacher.k);
}

// loss = sum of the row losses (/ count), one workgroup, in a fixed order.
__global__ __launch_bounds__(kRowThreads) void k_loss_sum(const float* row_loss, int64_t rows, const int* count,
                                                          float* loss) {
  __shared__ double lds[kRowThreads / 64];
  double s = 0.;
  for (int64_t r = threadIdx.x; r < rows; r += kRowThreads) s += row_loss[r];
  s = block_reduce(s, lds, [](double a, double b) { return a + b; });
  if (threadIdx.x == 0) *loss = (float)(count ? s / (*count > 0 ? *count : 1) : s);
}

__global__ void k_zero_word(int* p) { *p = 0; }

}  // namespace mec
