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
#include "mec_vec.h"

namespace mec {

constexpr float kLn2 = 0.69314718055994531f;

// Row r starts at (r / inner) * outer_stride + (r % inner) * inner_stride
// elements (64 bits: a matrix of logits passes 2^32 elements).
struct RowMap {
  int64_t inner, outer_stride, inner_stride;
  __device__ __forceinline__ int64_t operator()(int64_t r) const {
    if (inner == 1) return r * outer_stride;
    const uint32_t q = (uint32_t)r / (uint32_t)inner;  // (r < 2^23)
    return q * outer_stride + ((uint32_t)r - q * (uint32_t)inner) * inner_stride;
  }
};

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

// The wave's sum (largest), the same in every lane and in the same order on
// every run: six lane moves of the vector unit instead of trips to LDS.
template <class Op>
__device__ __forceinline__ float wave_all(float v, float none, Op op) {
  auto step = [&](auto ctrl, auto rows) {
    const int moved = __builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), decltype(ctrl)::value,
                                                  decltype(rows)::value, 0xf, false);
    v = op(v, __int_as_float(moved));
  };
  using std::integral_constant;
  step(integral_constant<int, 0xb1>{}, integral_constant<int, 0xf>{});   // lane ^ 1
  step(integral_constant<int, 0x4e>{}, integral_constant<int, 0xf>{});   // lane ^ 2
  step(integral_constant<int, 0x141>{}, integral_constant<int, 0xf>{});  // mirrored in 8 lanes
  step(integral_constant<int, 0x140>{}, integral_constant<int, 0xf>{});  // mirrored in 16
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // lane 15 of a row of 16 to the next
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // lane 31 to the upper half
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_total(float v) {
  return wave_all(v, 0.f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_most(float v) {
  return wave_all(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}

// t = (x - m) c as one fma with m c rounded beforehand.  The rounding of m c, below
// 2^-2, moves every t of the row alike and drops out of p and log p, which are formed
// from t.  Where m c is larger, up to fp32's end, the difference is taken first.
struct Reference {
  float m, c, mc;
  bool far;
  __device__ __forceinline__ Reference(float row_max, float scale) {
    m = row_max == -INFINITY ? 0.f : row_max;
    c = scale;
    mc = m * c;
    asm("" : "+v"(mc));  // one rounded number wherever it is used, not part of another fma
    far = !(fabsf(mc) < 4194304.f);
  }
  __device__ __forceinline__ float t(float x) const { return far ? 2.f * c * (0.5f * x - 0.5f * m) : fmaf(x, c, -mc); }
  // what to add to t of this one to have it relative to `to`
  __device__ __forceinline__ float shift(const Reference& to) const {
    if (far) return to.t(m);
    return to.far ? fmaf(-to.m, c, mc) : mc - to.mc;
  }
};

// ---- token log probabilities ----
//
// A row is cut into segments that a workgroup holds in registers: up to 8
// vectors of 16 bytes a thread.  A segment is read once; maximum, sums and the
// top k come from the registers.  Rows of more than one segment are joined by
// k_scores_join.

constexpr int kSegChunks = 8;

// Workgroups of a launch over all segments of all rows: neighbours are the
// segments of one row, then the next row's.  A row of workgroups of the grid
// holds `rows_x` rows (below 2^32 work-items).
struct SegmentGrid {
  int segments, len;
  uint32_t rows_x;
  __device__ __forceinline__ bool place(int64_t rows, int64_t& r, int& seg) const {
    const uint32_t q = blockIdx.x / (uint32_t)segments;
    seg = (int)(blockIdx.x - q * segments);
    r = (int64_t)blockIdx.y * rows_x + q;
    return r < rows;
  }
};
constexpr int kMaxSegments = 64;  // a lane each in the join

// A vector's words with -inf outside of its elements [lo, hi).
template <class T>
__device__ __forceinline__ typename Vec<T>::raw own_elements(typename Vec<T>::raw r, int lo, int hi) {
  constexpr uint32_t kInf = std::is_same<T, float>::value      ? 0xff800000u
                            : std::is_same<T, uint16_t>::value ? 0xff80ff80u
                                                               : 0xfc00fc00u;
  constexpr int kPer = 4 / sizeof(T);  // elements in a word
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (i * kPer + e >= lo && i * kPer + e < hi) mask |= (kPer == 1 ? ~0u : 0xffffu) << (16 * e);
    r[i] = (r[i] & mask) | (kInf & ~mask);
  }
  return r;
}

// Elements between the last 4-byte boundary and p.  Vectors begin on these: off
// them the loads take 1.35 times as long (8192 x 50001 bf16), while 16-byte
// boundaries make no difference (50002, 50004 against 50008).
template <class T>
__device__ __forceinline__ int misaligned(const T* p) {
  return (int)(((uintptr_t)p & 3) / sizeof(T));
}

// Elements [base, base + size) of a row of n that begins `shift` elements past a
// boundary: segment `seg` (size <= 0: none).
struct SegmentRange {
  int base, size;
  __device__ __forceinline__ SegmentRange(int seg, int len, int n, int shift) {
    const int from = seg * len - shift, to = from + len < n ? from + len : n;
    base = from > 0 ? from : 0;
    size = to - base;
  }
};

template <class T, int THREADS = kRowThreads>
struct Segment {
  static constexpr int N = Vec<T>::N, kChunk = THREADS * N;
  typename Vec<T>::raw v[kSegChunks];
  // elements; where the thread's first vector would begin; elements from the
  // boundary before the segment on
  int n, first, span;
  // The shape of a segment of `count` elements at p.  Vectors begin on boundaries
  // (misaligned), but for one that would begin before the segment or end after it,
  // which is moved into it.
  __device__ __forceinline__ void shape(const T* p, int count) {
    // (opaque: in a loop over segments the compiler else makes a copy of the code for
    // each number of vectors)
    count = __builtin_amdgcn_readfirstlane(count);
    asm volatile("" : "+s"(count));
    n = count;
    const int shift = n < N ? 0 : misaligned(p);
    first = (int)threadIdx.x * N - shift;
    span = n + shift;
  }
  // where chunk c's vector would begin, and where it does
  __device__ __forceinline__ int place(int c) const { return c * kChunk + first; }
  __device__ __forceinline__ int begin(int c) const {
    const int at = place(c) > 0 ? place(c) : 0;
    return n < N ? 0 : at < n - N ? at : n - N;
  }
  // n elements at p; with ONCE the elements that a moved vector shares with
  // another thread's are -inf in it.
  template <bool ONCE>
  __device__ __forceinline__ void load(const T* p, int count) {
    shape(p, count);
    if (n < N) {
      v[0] = load_raw(p, first == 0 ? n : 0);
      v[0] = own_elements<T>(v[0], 0, first == 0 ? n : 0);
      return;
    }
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c) {
      // (set in any case: a register set in one trip alone is kept through the next)
      if (c * kChunk < span)
        v[c] = *(const typename Vec<T>::raw*)(p + begin(c));
      else
        v[c] = own_elements<T>(v[c], 0, 0);
    }
    if constexpr (!ONCE) return;
    if (first < 0) v[0] = own_elements<T>(v[0], 0, N + first);
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c)
      if (c * kChunk < span && (c + 1) * kChunk > span) {
        const int lo = place(c) - begin(c);
        if (lo > 0) v[c] = own_elements<T>(v[c], lo, N);
      }
  }
  // chunk c's vector to a segment of the same shape
  template <bool PAST>
  __device__ __forceinline__ void store(T* p, int c, const float (&x)[N]) const {
    if (n >= N) {
      if (place(c) < n) store_vec<PAST>(p + begin(c), Vec<T>::pack(x));
    } else if (first == 0) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < n) put(p + e, x[e]);
    }
  }
  // the same after load<true>: elements of another thread are left to it
  template <bool PAST>
  __device__ __forceinline__ void store_own(T* p, int c, const float (&x)[N]) const {
    const int at = place(c);
    if (at >= 0 && at + N <= n) {
      store_vec<PAST>(p + at, Vec<T>::pack(x));
    } else if (at < n) {
      const int i0 = begin(c);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i0 + e >= at && i0 + e < at + N && i0 + e < n) put(p + i0 + e, x[e]);
    }
  }
  // Unpacked anew by every pass: what one pass unpacks is not kept for the next
  // (twice the registers, and spills).
  __device__ __forceinline__ void values(int c, float (&x)[N]) {
    asm volatile("" : "+v"(v[c]));
    Vec<T>::unpack(v[c], x);
  }
  // The largest element of each of the thread's vectors (not NaN), and of all.
  __device__ __forceinline__ float maxima(float (&most)[kSegChunks]) {
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c) {
      most[c] = -INFINITY;
      if (c * kChunk >= span) continue;
      float x[N];
      values(c, x);
#pragma unroll
      for (int e = 0; e < N; ++e) most[c] = fmaxf(most[c], x[e]);
      m = fmaxf(m, most[c]);
    }
    return m;
  }
  // f(element, its index) over the thread's elements that pred holds for, few,
  // all in vectors that look(vector) holds for.  Every lane goes to its own next
  // vector and its own next element: a wave takes as many steps as its lane with
  // the most, not one for each vector and element that any lane wants.
  template <class L, class P, class F>
  __device__ __forceinline__ void each_of(L look, P pred, F f) {
    uint32_t vectors = 0;
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c)
      if (place(c) < n && look(c)) vectors |= 1u << c;
#pragma unroll 1
    for (; vectors; vectors &= vectors - 1) {
      const int at = __ffs(vectors) - 1;
      typename Vec<T>::raw r = v[0];
#pragma unroll
      for (int c = 1; c < kSegChunks; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = at == c ? v[c][i] : r[i];
      float x[N];
      Vec<T>::unpack(r, x);
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) hits |= pred(x[e]) ? 1u << e : 0u;
      const int i0 = begin(at);
#pragma unroll 1
      for (; hits; hits &= hits - 1) {
        const int e = __ffs(hits) - 1;
        float y = x[0];
#pragma unroll
        for (int q = 1; q < N; ++q) y = e == q ? x[q] : y;
        if (i0 + e >= place(at) && i0 + e < place(at) + N && i0 + e < n) f(y, i0 + e);
      }
    }
  }
  // whether a vector of chunk c has -inf in place of another thread's elements
  __device__ __forceinline__ bool edge(int c) const {
    return (c == 0 && span != n) || ((c + 1) * kChunk > span && span % N != 0);
  }
  // f(element) over the thread's elements (and -inf in place of others'), in the
  // chunks with an edge g(element)
  template <class F, class G>
  __device__ __forceinline__ void each(F f, G g) {
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c) {
      if (c * kChunk >= span) break;
      if (place(c) >= n) continue;
      float x[N];
      values(c, x);
      if (edge(c)) {
#pragma unroll
        for (int e = 0; e < N; ++e) g(x[e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) f(x[e]);
      }
    }
  }
  // f(element) over the thread's elements (and -inf in place of others')
  template <class F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c) {
      if (c * kChunk >= span) break;
      if (place(c) >= n) continue;
      float x[N];
      values(c, x);
#pragma unroll
      for (int e = 0; e < N; ++e) f(x[e]);
    }
  }
};

// Of the keys that the wave's lanes hold through key(i), i < per_lane, all
// different: a number that exactly k of them reach.
template <class F>
__device__ __forceinline__ uint64_t kth_largest(int per_lane, int k, F key) {
  uint64_t cut = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const uint64_t trial = cut | (1ull << bit);
    int reach = 0;
    for (int i = 0; i < per_lane; ++i) reach += __popcll(__ballot(key(i) >= trial));
    if (reach >= k) {
      cut = trial;
      if (reach == k) break;
    }
  }
  return cut;
}

constexpr int kCandidates = 1024;

struct TopLds {
  float thread_max[kRowThreads];
  uint64_t found[kCandidates];
  int count, scan[kRowThreads / 64];
  float cut;
};

// After thread_max is there (and count is 0): by the first wave, a value that at
// least k elements of the segment reach: so many threads' maxima do.
__device__ __forceinline__ void top_cut(TopLds& l, int k) {
  constexpr int kPer = kRowThreads / 64;
  const int lane = threadIdx.x;
  uint32_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) key[i] = order_bits(l.thread_max[i * 64 + lane]);
  uint32_t cut = 0;
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t trial = cut | (1u << bit);
    int reach = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) reach += __popcll(__ballot(key[i] >= trial));
    if (reach >= k) {
      cut = trial;
      if (reach <= k + k / 4) break;
    }
  }
  // (0: too few threads have elements; as NaN it keeps nothing out)
  if (lane == 0) l.cut = key_value((uint64_t)cut << 32);
}

// The k largest of n elements at x, where more of them reach `cut` than there is
// room for (equal values, or a few threads with most of the large ones): the
// k-th largest value exactly, the elements above it, and the first of those equal
// to it.  Reads them again, from the cache; rare.
template <class T>
__device__ __attribute__((noinline)) void top_exactly(TopLds& l, const T* x, int n, int base, int k) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  auto count_from = [&](uint32_t from) {
    int c = 0;
    for (int i = tid; i < n; i += kRowThreads) c += order_bits(value(x[i])) >= from;
    for (int s = 32; s >= 1; s >>= 1) c += __shfl_xor(c, s, 64);
    __syncthreads();
    if (lane == 0) l.scan[w] = c;
    __syncthreads();
    return l.scan[0] + l.scan[1] + l.scan[2] + l.scan[3];
  };
  const float cut = l.cut;
  uint32_t kth = cut != cut ? 0u : order_bits(cut);  // reached by k at least
  if (kth == 0 || count_from(kth + 1) >= k) {
    kth = 0;
    for (int bit = 31; bit >= 0; --bit)
      if (count_from(kth | (1u << bit)) >= k) kth |= 1u << bit;
  }
  __syncthreads();
  if (tid == 0) l.count = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kRowThreads)
    if (order_bits(value(x[i])) > kth) l.found[atomicAdd(&l.count, 1)] = order_key(value(x[i]), base + i);
  __syncthreads();
  int have = l.count;
  for (int i0 = 0; i0 < n && have < k; i0 += kRowThreads) {
    const int i = i0 + tid;
    const bool mine = i < n && order_bits(value(x[i])) == kth;
    const uint64_t mask = __ballot(mine);
    __syncthreads();
    if (lane == 0) l.scan[w] = __popcll(mask);
    __syncthreads();
    int at = have + __popcll(mask & ((1ull << lane) - 1));
    for (int q = 0; q < w; ++q) at += l.scan[q];
    if (mine && at < k) l.found[at] = order_key(value(x[i]), base + i);
    have += l.scan[0] + l.scan[1] + l.scan[2] + l.scan[3];
  }
  __syncthreads();
  if (tid == 0) l.count = k;
  __syncthreads();
}

// The k largest of the segment (and perhaps others), keys with indexes from
// `base`, at found[0 .. count) in no order; k <= the segment's elements.  Only
// vectors whose maximum reaches the cut are looked into, all where there is a NaN.
template <class T>
__device__ __forceinline__ void top_collect(TopLds& l, Segment<T>& v, const float (&most)[kSegChunks], bool nan,
                                            const T* x, int base, int k) {
  const float cut = l.cut;
  v.each_of([&](int c) { return nan || !(most[c] < cut); }, [&](float f) { return !(f < cut); },
            [&](float f, int i) {
              const int at = atomicAdd(&l.count, 1);
              if (at < kCandidates) l.found[at] = order_key(f, base + i);
            });
  __syncthreads();
  if (l.count > kCandidates) top_exactly(l, x, v.n, base, k);
}

struct ScoresOut {
  float* log_probs;
  float* entropy;
  int64_t* top_tokens;
  float* top_log_probs;
  float* stats;  // m, S; or null
};

// One row's result from its sums.
struct RowResult {
  Reference ref;
  float s, ls, inv_t;
  __device__ __forceinline__ RowResult(const Reference& r, float sum, float it)
      : ref(r), s(sum), ls(logf(sum)), inv_t(it) {}
  __device__ __forceinline__ float log_prob(float x) const {
    if (s == 0.f) return -INFINITY;
    const float t = ref.t(x);  // (log2's units pass fp32's range before the result does)
    return (t > -1e30f ? kLn2 * t : scaled_difference(x, ref.m, inv_t)) - ls;
  }
  __device__ __forceinline__ float entropy(float u) const { return s == 0.f ? 0.f : ls - kLn2 * (u / s); }
};

__device__ __forceinline__ void write_ignored(const ScoresOut& out, int64_t r, int64_t rows, int k, int tid,
                                              int threads) {
  if (tid == 0) {
    out.log_probs[r] = 0.f, out.entropy[r] = 0.f;
    if (out.stats) out.stats[r] = 0.f, out.stats[rows + r] = 0.f;
  }
  for (int j = tid; j < k; j += threads) out.top_tokens[r * k + j] = -1, out.top_log_probs[r * k + j] = 0.f;
}

// One workgroup per segment of a row.  With one segment the row's results, else
// parts[row][seg] = (m, S, U) and the segment's top k keys.
//
// Bound by the vector unit, busy 93% of the time (98% with top tokens), with the read
// close behind: 10 instructions a value (14 with 32 top tokens), the exponential for
// two: an unpack twice (maximum, sums), half a maximum, three fma-like operations and
// what goes round them.  256 threads and 8 vectors each: 51 to 67 registers, so that
// seven or eight workgroups share a CU and one's sums hide the others' loads.  8192 x
// 49408 bf16 in 138 us (5.9 TB/s); with the 32 top tokens, 4096 x 131072 bf16, a tenth
// of them ignored, 190 us (5.1 TB/s).
template <class T, bool TOP>
__global__ __launch_bounds__(kRowThreads) void k_scores(const T* logits, RowMap map, int n, Tokens tokens,
                                                        int64_t ignore, float inv_t, int k, ScoresOut out,
                                                        int64_t rows, SegmentGrid grid, float4* parts,
                                                        uint64_t* part_top) {
  constexpr int kWaves = kRowThreads / 64;
  __shared__ float wave_max[kWaves], wave_s[kWaves], wave_u[kWaves];
  __shared__ std::conditional_t<TOP, TopLds, char> top;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float c = inv_t * (1.f / kLn2);
  const int segments = grid.segments, len = grid.len;
  int64_t r;
  int seg;
  if (!grid.place(rows, r, seg)) return;
  const int64_t item = r * segments + seg;
  const int64_t tok = tokens[r];
  if (tok == ignore) {
    if (segments == 1) write_ignored(out, r, rows, k, tid, kRowThreads);
    return;
  }
  const T* x = logits + map(r);
  const SegmentRange range(seg, len, n, misaligned(x));
  const int base = range.base;
  if (range.size <= 0) {  // (the last one, of a row that needs one less)
    if (tid == 0) parts[item] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    for (int i = tid; i < k; i += kRowThreads) part_top[item * k + i] = 0;
    return;
  }
  x += base;
  Segment<T> v;
  v.template load<true>(x, range.size);
  float most[kSegChunks];
  float m = v.maxima(most);
  if constexpr (TOP) {
    top.thread_max[tid] = m;
    if (tid == 0) top.count = 0;
  }
  m = wave_most(m);
  if (lane == 0) wave_max[w] = m;
  __syncthreads();
  m = wave_max[0];
  for (int i = 1; i < kWaves; ++i) m = fmaxf(m, wave_max[i]);
  const int kk = TOP ? (k < v.n ? k : v.n) : 0;
  if constexpr (TOP) {
    if (w == 0) top_cut(top, kk);
  }
  const Reference ref(m, c);
  float s = 0.f, u = 0.f;
  auto careful = [&](float f) {
    const float t = ref.t(f);
    const float e = fast_exp2(t);
    s += e;
    // (2^t is 0 below -200, where t may be -inf)
    u = fmaf(e, fmaxf(t, -200.f), u);
  };
  // Where no t is -inf the plain form does, with one operation in eleven less (138
  // against 162 us for 8192 x 50008 bf16); a wave that meets one has a U of NaN and
  // starts again.
  if (!ref.far) {
    v.each(
        [&](float f) {
          const float t = fmaf(f, c, -ref.mc), e = fast_exp2(t);
          s += e;
          u = fmaf(e, t, u);
        },
        careful);
    s = wave_total(s);
    u = wave_total(u);
  }
  if (ref.far || u != u) {
    s = u = 0.f;
    v.each(careful);
    s = wave_total(s);
    u = wave_total(u);
  }
  if (lane == 0) wave_s[w] = s, wave_u[w] = u;
  __syncthreads();
  s = u = 0.f;
  for (int i = 0; i < kWaves; ++i) s += wave_s[i], u += wave_u[i];
  if constexpr (TOP) top_collect(top, v, most, s != s, x, base, kk);
  if (tid == 0) {
    if (segments == 1) {
      const RowResult row(ref, s, inv_t);
      out.log_probs[r] = tok >= 0 && tok < n ? row.log_prob(value(x[tok])) : NAN;
      out.entropy[r] = row.entropy(u);
      if (out.stats) out.stats[r] = ref.m, out.stats[rows + r] = s;
    } else {
      parts[item] = make_float4(m, s, u, 0.f);
    }
  }
  if constexpr (TOP) {
    const int count = top.count;
    for (int i = tid; i < count; i += kRowThreads) {
      const uint64_t key = top.found[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += top.found[j] > key;
      if (rank >= kk) continue;
      if (segments == 1) {
        out.top_tokens[r * k + rank] = key_index(key);
        out.top_log_probs[r * k + rank] = RowResult(ref, s, inv_t).log_prob(key_value(key));
      } else {
        part_top[item * k + rank] = key;
      }
    }
    if (segments > 1)
      for (int i = kk + tid; i < k; i += kRowThreads) part_top[item * k + i] = 0;
  }
}

constexpr int kJoinThreads = 256;
constexpr int kJoinRank = 256;  // above it, a search for the k-th key is shorter than ranking all

// One workgroup per row: its segments' sums, a lane of the first wave each, and
// the k largest of their top keys (all different: exactly k reach the k-th).
// Bound by the latency of four dependent reads: 4096 rows of 8 lists of 32 keys
// 11 us, one row of 64 lists of 20 keys 7 us (all keys ranked: 99 us).
template <class T>
__global__ __launch_bounds__(kJoinThreads) void k_scores_join(const T* logits, RowMap map, int n, Tokens tokens,
                                                              int64_t ignore, float inv_t, int k, ScoresOut out,
                                                              int64_t rows, int segments, const float4* parts,
                                                              const uint64_t* part_top) {
  extern __shared__ uint64_t keys[];  // segments * k
  __shared__ uint64_t cut_at;
  __shared__ int kept;
  __shared__ float2 sums;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t tok = tokens[r];
  if (tok == ignore) {
    write_ignored(out, r, rows, k, tid, kJoinThreads);
    return;
  }
  const int count = segments * k;
  part_top += r * count;
  const float c = inv_t * (1.f / kLn2);
  const uint64_t early = tid < count ? part_top[tid] : 0;  // on its way while the cut is found
  if (tid < 64) {
    const float at = tok >= 0 && tok < n ? value(logits[map(r) + tok]) : 0.f;
    const float4 p = lane < segments ? parts[r * segments + lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
    // The lists are in order: if q lists have their p-th key at or above a cut,
    // p q keys are.  The cut is the q-th of the p-th keys, p q >= k.
    const int p_th = k ? (k + segments - 1) / segments : 1, q_th = k ? (k + p_th - 1) / p_th : 1;
    const uint64_t head = k && lane < segments ? part_top[lane * k + p_th - 1] : 0;
    float m = p.x;
    m = wave_most(m);
    const Reference ref(m, c);
    // (S = 0: nothing of the segment can occur, and its shift may be -inf)
    const float shift = Reference(p.x, c).shift(ref), scale = fast_exp2(shift);
    const float s = wave_total(p.y == 0.f ? 0.f : p.y * scale);
    const float u = wave_total(p.y == 0.f ? 0.f : scale * fmaf(p.y, fmaxf(shift, -200.f), p.z));
    const RowResult row(ref, s, inv_t);
    if (lane == 0) {
      out.log_probs[r] = tok >= 0 && tok < n ? row.log_prob(at) : NAN;
      out.entropy[r] = row.entropy(u);
      if (out.stats) {
        out.stats[r] = ref.m;
        out.stats[rows + r] = s;
      }
      sums = make_float2(ref.m, s);
      kept = 0;
    }
    if (k) {
      int above = 0;
      for (int i = 0; i < segments; ++i) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(head >> 32), i) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)head, i);
        above += other > head || (other == head && i < lane);
      }
      // (lists shorter than k end in 0; keys are not 0)
      if (lane < segments && above == q_th - 1) cut_at = head ? head : 1;
    }
  }
  if (k == 0) return;
  __syncthreads();
  uint64_t cut = cut_at;
  uint64_t* found = keys;
  if (early >= cut) found[atomicAdd(&kept, 1)] = early;
#pragma unroll 4
  for (int i = tid + kJoinThreads; i < count; i += kJoinThreads) {
    const uint64_t key = part_top[i];
    if (key >= cut) found[atomicAdd(&kept, 1)] = key;
  }
  __syncthreads();
  int have = kept;
  if (have > kJoinRank) {
    // the k-th key itself, and the keys from it on to the front, by the first wave
    if (tid < 64) {
      cut = kth_largest((have + 63) / 64, k, [&](int i) { return i * 64 + lane < have ? found[i * 64 + lane] : 0; });
      int at = 0;
      for (int i0 = 0; i0 < have; i0 += 64) {
        const uint64_t key = i0 + lane < have ? found[i0 + lane] : 0;
        const uint64_t mask = __ballot(key >= cut);
        if (key >= cut) found[at + __popcll(mask & ((1ull << lane) - 1))] = key;
        at += __popcll(mask);
      }
    }
    have = k;
    __syncthreads();
  }
  const RowResult row(Reference(sums.x, c), sums.y, inv_t);
  for (int i = tid; i < have; i += kJoinThreads) {
    const uint64_t key = found[i];
    int rank = 0;
    for (int j = 0; j < have; ++j) rank += found[j] > key;
    if (rank >= k) continue;
    out.top_tokens[r * k + rank] = key_index(key);
    out.top_log_probs[r * k + rank] = row.log_prob(key_value(key));
  }
}

// dx_v = (1/T) (g_l (1[v = tok] - p_v) - g_h p_v (log p_v + entropy)), which is
// 2^t (a + b t) but for the token's own term.  One workgroup per segment of a row; a
// vector that is moved into the segment (Segment::begin) stores values that another
// thread stores as well, the same ones.  Bound by memory: 8192 x 49408 bf16, a quarter
// of the rows ignored, 245 us for 0.61 GB read and 0.81 GB written (5.8 TB/s, some of
// the reads from the cache).
template <class T, bool PAST>
__global__ __launch_bounds__(kRowThreads) void k_scores_grad(const T* logits, RowMap map, int n, Tokens tokens,
                                                             int64_t ignore, float inv_t, const float* stats,
                                                             const float* entropy, const float* g_log_probs,
                                                             const float* g_entropy, T* dx, int64_t rows,
                                                             SegmentGrid grid) {
  constexpr int N = Vec<T>::N;
  const int len = grid.len;
  int64_t r;
  int seg;
  if (!grid.place(rows, r, seg)) return;
  // the last rows first: what the forward read last is still cached
  r = rows - 1 - r;
  const int64_t tok = tokens[r];
  const T* x0 = logits + map(r);
  const SegmentRange range(seg, len, n, misaligned(x0));
  const int base = range.base;
  if (range.size <= 0) return;
  T* y = dx + r * n + base;
  const float s = stats[rows + r];
  const bool none = tok == ignore || s == 0.f, bad = tok < 0 || tok >= n;
  Segment<T> v;
  if (none)
    v.shape(x0 + base, range.size);
  else
    v.template load<false>(x0 + base, range.size);
  const Reference ref(stats[r], inv_t * (1.f / kLn2));
  const float ls = logf(s), gh = g_entropy ? g_entropy[r] : 0.f;
  float gl = g_log_probs ? g_log_probs[r] : 0.f;
  if (bad && gl != 0.f) gl = NAN;  // (the entropy does not depend on the token)
  // e (a + b t) = -(1/T) p (g_l + g_h (log p + entropy))
  const float f = none ? 0.f : -inv_t / s, a = f * (gl + gh * (entropy[r] - ls)), b = f * gh * kLn2;
  const int at = (int)(bad ? 0 : tok) - base;
#pragma unroll
  for (int c = 0; c < kSegChunks; ++c) {
    if (c * Segment<T>::kChunk >= v.span) break;
    float x[N];
    if (none) {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = 0.f;
    } else {
      v.values(c, x);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float t = ref.t(x[e]);
        x[e] = fast_exp2(t) * fmaf(b, fmaxf(t, -200.f), a);
      }
      const int own = at - v.begin(c);
      if (own >= 0 && own < N) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] += e == own ? gl * inv_t : 0.f;
      }
    }
    v.template store<PAST>(y, c, x);
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

// Which rows have a teacher, and how many of each workgroup's.
struct TeacherRows {
  int* some;    // [rows]
  int* counts;  // [groups]
  int groups, rows_each;
  // by one wave, in every lane
  __device__ __forceinline__ int total() const {
    int c = 0;
    for (int i = threadIdx.x & 63; i < groups; i += 64) c += counts[i];
    for (int i = 32; i >= 1; i >>= 1) c += __shfl_xor(c, i, 64);
    return c;
  }
};
constexpr int kTeacherThreads = 256, kTeacherRows = 16, kTeacherGroups = 1024;

__global__ __launch_bounds__(kTeacherThreads) void k_teacher_rows(Teacher t, int64_t rows, TeacherRows out) {
  __shared__ int has[kTeacherRows];
  __shared__ int count;
  const int tid = threadIdx.x;
  if (tid == 0) count = 0;
  const int64_t first = (int64_t)blockIdx.x * out.rows_each;
  const int64_t end = first + out.rows_each < rows ? first + out.rows_each : rows;
  for (int64_t r0 = first; r0 < end; r0 += kTeacherRows) {
    const int n = end - r0 < kTeacherRows ? (int)(end - r0) : kTeacherRows;
    if (tid < kTeacherRows) has[tid] = 0;
    __syncthreads();
    const int entries = n * t.k;
#pragma unroll 4
    for (int i = tid; i < entries; i += kTeacherThreads) {
      const int64_t tok = t.tokens[r0 * t.k + i];
      const float z = t.logit(r0 * t.k + i);
      if (tok >= 0 && z != -INFINITY) has[(uint32_t)i / (uint32_t)t.k] = 1;
    }
    __syncthreads();
    if (tid < n) {
      out.some[r0 + tid] = has[tid];
      if (has[tid]) atomicAdd(&count, 1);
    }
  }
  __syncthreads();
  if (tid == 0) out.counts[blockIdx.x] = count;
}

// One row's teacher in shared memory: q, log q and the tokens (-1: none).
struct TeacherRow {
  float *q, *log_q;
  int* tok;
  int k;
  __device__ __forceinline__ TeacherRow(float* lds, int entries)
      : q(lds), log_q(lds + entries), tok((int*)lds + 2 * entries), k(entries) {}
  // By one wave; true if a token lies past the vocabulary.
  __device__ __forceinline__ bool load(const Teacher& t, int64_t r, int n, float inv_t) {
    const int lane = threadIdx.x & 63;
    const float c = inv_t * (1.f / kLn2);
    float m = -INFINITY;
    bool bad = false;
    for (int j = lane; j < k; j += 64) {
      const int64_t v = t.tokens[r * k + j];
      const float z = v < 0 ? -INFINITY : t.logit(r * k + j);
      bad |= v >= n;
      tok[j] = v < 0 || v >= n ? -1 : (int)v;
      log_q[j] = z;
      m = fmaxf(m, z);
    }
    m = wave_most(m);
    const Reference ref(m, c);
    float s = 0.f;
    for (int j = lane; j < k; j += 64) s += fast_exp2(ref.t(log_q[j]));
    s = wave_total(s);
    const float ls = logf(s);
    for (int j = lane; j < k; j += 64) {
      const float z = ref.t(log_q[j]);
      q[j] = s == 0.f ? 0.f : fast_exp2(z) / s;
      log_q[j] = kLn2 * z - ls;
    }
    return __any(bad);
  }
  // sum_j q_j (log q_j - log p_j) by the wave that loaded it; x: the row's logits
  template <class T>
  __device__ __forceinline__ float divergence(const T* x, const Reference& ref, float s, float inv_t) const {
    const RowResult row(ref, s, inv_t);
    float loss = 0.f;
    for (int j = threadIdx.x & 63; j < k; j += 64)
      if (!(q[j] == 0.f) && tok[j] >= 0) loss += q[j] * (log_q[j] - row.log_prob(value(x[tok[j]])));
    return wave_total(loss);
  }
  // After y = g p over [base, base + count) of a row: y at the teacher's tokens
  // there, each by one thread from all its entries.
  template <class T>
  __device__ __forceinline__ void subtract(const T* x, T* y, int base, int count, const Reference& ref, float gs,
                                           float g) const {
    for (int j = threadIdx.x; j < k; j += blockDim.x) {
      const int v = tok[j];
      if (v < base || v >= base + count) continue;
      float sum = 0.f;
      for (int i = 0; i < k; ++i) sum += tok[i] == v ? q[i] : 0.f;
      put(y + v, fast_exp2(ref.t(value(x[v]))) * gs - g * sum);
    }
  }
};

// What the backward has to know of a row: m and S; S < 0: the row has no
// teacher, S = 0: nothing can occur (both: no gradient), NaN: no result.
struct DistillState {
  float* m;
  float* s;
};

// Loss and gradient (for grad_output 1) of a row by one workgroup.  With ONE the
// row is one segment and stays in registers from its only read to the gradient's
// write.  Of a longer row the last segment stays in registers, the one before it in
// LDS and the one before that in registers again (192 KB of a row with 512 threads,
// 384 KB with 1024); what is left is read a second time.  Bound by memory (the vector
// unit is busy 75 to 82% of the time): with ONE or 512 threads two or more workgroups
// share a CU, so that one reads while the other writes (8192 x 49408 bf16, a quarter
// without a teacher: 288 us, 4.9 TB/s; 8192 x 70001: 512 us, 4.5 TB/s; 4096 x 200000,
// half of the row read twice: 2.5 GB past L2 and 1.7 written in 705 us, 4.6 TB/s
// without the second reads); 1024 threads with more than a segment have the CU to
// themselves (1024 x 400000 bf16: 412 us, 4.0 TB/s).  Which of the two: row_shape.
template <class T, int THREADS, bool ONE, bool PAST>
__global__ __launch_bounds__(THREADS, ONE ? 1 : 4) void k_distill_row(
    const T* logits, RowMap map, int n, Teacher teacher, float inv_t, float scale, TeacherRows have, int mean,
    float* row_loss, DistillState state, T* dx, int segments, int len) {
  constexpr int N = Vec<T>::N, kWaves = THREADS / 64;
  extern __shared__ float teacher_lds[];
  __shared__ float2 wave_sums[kWaves];
  __shared__ int bad_row, count;
  __shared__ typename Vec<T>::raw held[ONE ? 1 : kSegChunks][ONE ? 1 : THREADS];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const T* x = logits + map(r);
  T* y = dx + r * n;
  Segment<T, THREADS> v;
  [[maybe_unused]] typename Vec<T>::raw kept[ONE ? 1 : kSegChunks];
  // (the first segment is the short one, up to a boundary: the others fill the registers)
  const int shift = misaligned(x);
  const int first_size = ONE ? n : (n - (segments - 1) * len + shift + N - 1) / N * N - shift;
  auto seg_base = [&](int i) { return i ? first_size + (i - 1) * len : 0; };
  auto seg_size = [&](int i) { return (i < segments - 1 ? seg_base(i + 1) : n) - seg_base(i); };
  auto each_segment = [&](auto f) {  // f(segment, its first element, its size)
    if constexpr (ONE)
      f(0, 0, n);
    else
      for (int i = 0; i < segments; ++i) f(i, seg_base(i), seg_size(i));
  };
  if (!have.some[r]) {
    if (tid == 0) row_loss[r] = 0.f, state.m[r] = 0.f, state.s[r] = -1.f;
    each_segment([&](int, int base, int size) {
      v.shape(x + base, size);
      const float zero[N] = {};
#pragma unroll
      for (int c = 0; c < kSegChunks; ++c)
        if (c * Segment<T, THREADS>::kChunk < v.span) v.template store<PAST>(y + base, c, zero);
    });
    return;
  }
  TeacherRow row(teacher_lds, teacher.k);
  const float c_log2 = inv_t * (1.f / kLn2);
  // each wave's own largest and sum: no waiting for others until all is read
  float m = -INFINITY, s = 0.f;
  each_segment([&](int i, int base, int size) {
    v.template load<true>(x + base, size);
    if (i == 0 && w == 0) {
      const bool bad = row.load(teacher, r, n, inv_t);
      if (lane == 0) bad_row = bad;
    }
    if (i == 0 && w == 1) {
      const int rows_in = mean ? have.total() : 1;
      if (lane == 0) count = rows_in;
    }
    float most[kSegChunks];
    const float m_old = m;
    m = fmaxf(m, wave_most(v.maxima(most)));
    const Reference ref(m, c_log2);
    if (!ONE && i > 0 && s != 0.f) s *= fast_exp2(Reference(m_old, c_log2).shift(ref));
    v.each([&](float f) { s += fast_exp2(ref.t(f)); });
    if constexpr (!ONE) {
      if (i == segments - 2) {
#pragma unroll
        for (int c = 0; c < kSegChunks; ++c)
          if (c * Segment<T, THREADS>::kChunk < v.span) held[c][tid] = v.v[c];
      } else if (i == segments - 3) {
#pragma unroll
        for (int c = 0; c < kSegChunks; ++c) kept[c] = v.v[c];
      }
    }
  });
  s = wave_total(s);
  if (lane == 0) wave_sums[w] = make_float2(m, s);
  __syncthreads();
  m = wave_sums[0].x;
#pragma unroll
  for (int i = 1; i < kWaves; ++i) m = fmaxf(m, wave_sums[i].x);
  const Reference ref(m, c_log2);
  s = 0.f;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const float2 p = wave_sums[i];
    s += p.y == 0.f ? 0.f : p.y * fast_exp2(Reference(p.x, c_log2).shift(ref));
  }
  const bool bad = bad_row;
  const float g = scale / (inv_t * fmaxf((float)count, 1.f)), gs = bad ? NAN : s == 0.f ? 0.f : g / s;
  auto write = [&](int base) {
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c) {
      if (c * Segment<T, THREADS>::kChunk >= v.span) break;
      float f[N];
      v.values(c, f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = fast_exp2(ref.t(f[e])) * gs;
      v.template store_own<PAST>(y + base, c, f);
    }
  };
  if constexpr (ONE) {
    write(0);
  } else {
    write(seg_base(segments - 1));
    for (int i = segments - 2; i >= 0; --i) {
      const int base = seg_base(i), size = seg_size(i);
      if (i == segments - 2) {
        v.shape(x + base, size);
#pragma unroll
        for (int c = 0; c < kSegChunks; ++c)
          if (c * Segment<T, THREADS>::kChunk < v.span) v.v[c] = held[c][tid];
      } else if (i == segments - 3) {
        v.shape(x + base, size);
#pragma unroll
        for (int c = 0; c < kSegChunks; ++c) v.v[c] = kept[c];
      } else {
        v.template load<true>(x + base, size);
      }
      write(base);
    }
  }
  if (w == 0) {
    const float loss = row.divergence(x, ref, s, inv_t);
    if (lane == 0) {
      row_loss[r] = bad ? NAN : loss * (scale / (inv_t * inv_t));
      state.m[r] = ref.m;
      state.s[r] = bad ? NAN : s;
    }
  }
  if (bad || s == 0.f) return;
  __syncthreads();
  row.subtract(x, y, 0, n, ref, gs, g);
}

// m and S of a segment: the loss without its gradient (1003 x 32001 fp16 14 us,
// 4096 x 200000 bf16 320 us, 5.1 TB/s).
template <class T>
__global__ __launch_bounds__(kRowThreads) void k_distill_sums(const T* logits, RowMap map, int n, float inv_t,
                                                              const int* some, int64_t rows, SegmentGrid grid,
                                                              float2* parts) {
  constexpr int kWaves = kRowThreads / 64;
  __shared__ float wave_max[kWaves], wave_s[kWaves];
  int64_t r;
  int seg;
  if (!grid.place(rows, r, seg)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (!some[r]) return;
  const T* x = logits + map(r);
  const SegmentRange range(seg, grid.len, n, misaligned(x));
  if (range.size <= 0) {  // (the last one, of a row that needs one less)
    if (tid == 0) parts[r * grid.segments + seg] = make_float2(-INFINITY, 0.f);
    return;
  }
  Segment<T> v;
  v.template load<true>(x + range.base, range.size);
  float m = -INFINITY;
  v.each([&](float f) { m = fmaxf(m, f); });
  m = wave_most(m);
  if (lane == 0) wave_max[w] = m;
  __syncthreads();
  m = wave_max[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) m = fmaxf(m, wave_max[i]);
  const Reference ref(m, inv_t * (1.f / kLn2));
  float s = 0.f;
  v.each([&](float f) { s += fast_exp2(ref.t(f)); });
  s = wave_total(s);
  if (lane == 0) wave_s[w] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += wave_s[i];
    parts[r * grid.segments + seg] = make_float2(m, s);
  }
}

// A row's m, S and loss from its segments' sums, a lane each: one wave per row.
template <class T>
__global__ __launch_bounds__(64) void k_distill_join(const T* logits, RowMap map, int n, Teacher teacher, float inv_t,
                                                     float scale, const int* some, const float2* parts, int segments,
                                                     float* row_loss, DistillState state) {
  extern __shared__ float teacher_lds[];
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x;
  if (!some[r]) {
    if (lane == 0) row_loss[r] = 0.f, state.m[r] = 0.f, state.s[r] = -1.f;
    return;
  }
  TeacherRow row(teacher_lds, teacher.k);
  const float2 p = lane < segments ? parts[r * segments + lane] : make_float2(-INFINITY, 0.f);
  const bool bad = row.load(teacher, r, n, inv_t);
  float m = p.x;
  m = wave_most(m);
  const float c = inv_t * (1.f / kLn2);
  const Reference ref(m, c);
  const float s = wave_total(p.y == 0.f ? 0.f : p.y * fast_exp2(Reference(p.x, c).shift(ref)));
  __syncthreads();
  const float loss = row.divergence(logits + map(r), ref, s, inv_t);
  if (lane == 0) {
    row_loss[r] = bad ? NAN : loss * (scale / (inv_t * inv_t));
    state.m[r] = ref.m;
    state.s[r] = bad ? NAN : s;
  }
}

// dx from the rows' m and S.  grad_output: one number, or one for each row.  With
// `made` dx holds the gradient for grad_output 1, and only another one makes it anew
// (few workgroups then, each for many segments).
// Bound by memory: 1003 x 32001 fp16 21 us.
template <class T, bool PAST>
__global__ __launch_bounds__(kRowThreads) void k_distill_grad(const T* logits, RowMap map, int n, Teacher teacher,
                                                              float inv_t, float scale, const int* count,
                                                              DistillState state, const float* grad_output,
                                                              int per_row, int made, T* dx, int64_t rows, int len,
                                                              int segments) {
  constexpr int N = Vec<T>::N;
  extern __shared__ float teacher_lds[];
  if (made && *grad_output == 1.f) return;
  const int tid = threadIdx.x;
  const float rows_in = count ? fmaxf((float)*count, 1.f) : 1.f;
  const uint32_t items = (uint32_t)rows * segments;  // (< 2^29)
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t q = item / segments, r = (uint32_t)rows - 1 - q;  // the last ones first: they are still cached
    const T* x = logits + map(r);
    const SegmentRange range((int)(item - q * segments), len, n, misaligned(x));
    const int base = range.base, size = range.size;
    if (size <= 0) continue;
    T* y = dx + (int64_t)r * n;
    const float s = state.s[r];
    const bool none = s <= 0.f;
    Segment<T> v;
    if (none) {
      v.shape(x + base, size);
      const float zero[N] = {};
#pragma unroll
      for (int c = 0; c < kSegChunks; ++c)
        if (c * Segment<T>::kChunk < v.span) v.template store<PAST>(y + base, c, zero);
      continue;
    }
    v.template load<false>(x + base, size);
    TeacherRow row(teacher_lds, teacher.k);
    if (tid < 64) row.load(teacher, r, n, inv_t);
    const Reference ref(state.m[r], inv_t * (1.f / kLn2));
    const float g = grad_output[per_row ? r : 0] * scale / (inv_t * rows_in), gs = g / s;
#pragma unroll
    for (int c = 0; c < kSegChunks; ++c) {
      if (c * Segment<T>::kChunk >= v.span) break;
      float f[N];
      v.values(c, f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = fast_exp2(ref.t(f[e])) * gs;
      v.template store<PAST>(y + base, c, f);
    }
    __syncthreads();
    if (s == s) row.subtract(x, y, base, size, ref, gs, g);
    __syncthreads();
  }
}

// loss = sum of the row losses (/ the rows that have a teacher, noted in *count for
// the backward), one workgroup, in a fixed order.
constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void k_loss_sum(const float* row_loss, int64_t rows, TeacherRows have,
                                                          int mean, int* count, float* loss) {
  __shared__ double lds[kSumThreads / 64];
  double s = 0.;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < rows; r += kSumThreads) s += row_loss[r];
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int rows_in = mean ? have.total() : 1;
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSumThreads / 64; ++w) s += lds[w];
    *loss = (float)(s / (rows_in > 0 ? rows_in : 1));
    *count = rows_in;
  }
}

}  // namespace mec
