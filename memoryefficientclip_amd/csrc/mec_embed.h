// Scaled token embedding: y_t = scale W[tok_t], and its gradient
// dW_v = scale sum_{t: tok_t = v} dy_t.
//
// The gradient sorts the tokens (stable, so that a token's positions stay in
// order), sums long runs of one token in pieces, and then writes every row of
// dW once: no atomics, sums in fp32 in an order that depends on the tokens alone.
#pragma once
#include "mec_vocab.h"

namespace mec {

// Where the vector of a row of d elements begins that a lane takes for column
// `col`: one that would pass the end is the last one that does not (two lanes
// then do the same for the columns they share).  n: its elements, 0 for none.
template <int N>
__device__ __forceinline__ int vec_begin(int col, int d, int& n) {
  n = col >= d ? 0 : d < N ? d : N;
  return d < N || col < d - N ? col : d - N;
}

// scale * v in 32 bits, to be rounded after: not contracted with the rounding
// into one instruction that rounds the exact product to 16 bits.
__device__ __forceinline__ float scaled(float scale, float v) {
  float s = scale * v;
  asm("" : "+v"(s));
  return s;
}

constexpr int kEmbedThreads = 256;
constexpr int kEmbedTokens = 4;  // rows in flight per lane group

// A group of 2^lg lanes takes a token's row, kEmbedTokens rows at a time.  A
// token outside [0, vocab) gives a row of NaN.  Bound by memory: 524288 rows of 1024
// bf16 in 300 us (1.07 GB written; as much gathered, 0.47 GB of it past L2), 78848
// rows of 768 in 37 us.
template <class T, bool PAST>
__global__ __launch_bounds__(kEmbedThreads) void k_embed(Tokens tokens, int64_t n, const T* weight, int64_t ldw,
                                                         int64_t vocab, int d, int lg, float scale, T* out) {
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x & ((1 << lg) - 1);
  const int groups = kEmbedThreads >> lg;
  const int64_t t0 = (int64_t)blockIdx.x * groups * kEmbedTokens + (threadIdx.x >> lg);
  int64_t tok[kEmbedTokens];
#pragma unroll
  for (int i = 0; i < kEmbedTokens; ++i) {
    const int64_t t = t0 + i * groups;
    tok[i] = t < n ? tokens[t] : -1;
    if (tok[i] >= vocab) tok[i] = -1;
  }
  for (int col0 = lane * N; col0 < d; col0 += N << lg) {
    int n_col;
    const int col = vec_begin<N>(col0, d, n_col);
    float v[kEmbedTokens][N];
#pragma unroll
    for (int i = 0; i < kEmbedTokens; ++i) {
      if (tok[i] >= 0) {
        load_row(weight + tok[i] * ldw + col, n_col, v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[i][e] = NAN;
      }
    }
#pragma unroll
    for (int i = 0; i < kEmbedTokens; ++i) {
      const int64_t t = t0 + i * groups;
      if (t >= n) break;
#pragma unroll
      for (int e = 0; e < N; ++e) v[i][e] = scaled(scale, v[i][e]);
      store_row<PAST>(out + t * d + col, n_col, v[i]);
    }
  }
}

// ---- stable radix sort of (token, position) by token ----
//
// Digits of up to 9 bits.  The array is cut into tiles, a tile into a chunk of up
// to 8 x 64 pairs for each wave, which holds them in registers: lanes with the same
// digit find each other with ballots, and the first of them moves the wave's own
// counter of that digit.  A pass is two launches (tile counts, scatter; a third
// between them for more than 128 tiles); up to kSortOne pairs are sorted by one
// workgroup in one launch.  Two passes over 78848 pairs take 28 us, over 524288 48 us,
// over 5003 (one launch) 17 us: waiting, not moving, 16 bytes a pair and pass.

constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kSortBins = 512;
constexpr int kSortItems = 8;    // pairs per lane, at most
constexpr int kSortTiles = 128;  // up to here every workgroup reads all tiles' counts
constexpr int kSortOneThreads = 1024, kSortOne = kSortOneThreads * kSortItems;

struct SortShape {
  int64_t n;
  int items;  // pairs per lane
  int tiles;
  int vocab;  // tokens outside [0, vocab) and the padding get this key and come last
  int64_t padding;
};

struct SortSource {
  Tokens tokens;      // the first pass
  const uint2* pairs; // (key, position), the later ones; null in the first
};

struct SortOut {
  uint2* pairs;   // all passes but the last
  int* keys;      // the last
  int* positions;
  __device__ __forceinline__ void write(int64_t i, uint2 p) const {
    if (pairs) {
      pairs[i] = p;
    } else {
      keys[i] = (int)p.x;
      positions[i] = (int)p.y;
    }
  }
};

template <int THREADS>
struct SortLds {
  static constexpr int kWaves = THREADS / 64;
  int counters[kWaves][kSortBins];
  int scan[kWaves];
};

// Lanes of the wave with the same digit (of the active ones).
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool active) {
  uint64_t mask = __ballot(active);
  for (int b = 0; b < bits; ++b) {
    const uint64_t one = __ballot((digit >> b) & 1);
    mask &= (digit >> b) & 1 ? one : ~one;
  }
  return mask;
}

// A wave's pairs of a tile, in order: lane, then the next 64.
struct SortChunk {
  uint2 pair[kSortItems];
  int place[kSortItems];  // among the wave's pairs of the same digit
  int count;              // pairs
  __device__ __forceinline__ void load(const SortSource& src, const SortShape& s, int64_t tile) {
    const int lane = threadIdx.x & 63, per_wave = s.items * 64;
    const int64_t from = tile * (int64_t)(per_wave * kSortWaves) + (int64_t)(threadIdx.x >> 6) * per_wave;
    const int64_t left = s.n - from;
    count = left < 0 ? 0 : left < per_wave ? (int)left : per_wave;
#pragma unroll
    for (int b = 0; b < kSortItems; ++b) {
      const int i = b * 64 + lane;
      pair[b] = make_uint2(0, 0);
      if (i >= count) continue;
      if (src.pairs) {
        pair[b] = src.pairs[from + i];
      } else {
        const int64_t tok = src.tokens[from + i];
        const bool ok = tok >= 0 && tok < s.vocab && tok != s.padding;
        pair[b] = make_uint2(ok ? (uint32_t)tok : (uint32_t)s.vocab, (uint32_t)(from + i));
      }
    }
  }
  // Adds the digits to the wave's counters, and notes the places.
  __device__ __forceinline__ void rank(int shift, int bits, int* counters) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int b = 0; b < kSortItems; ++b) {
      if (b * 64 >= count) break;
      const bool active = b * 64 + lane < count;
      const uint32_t digit = (pair[b].x >> shift) & ((1u << bits) - 1);
      const uint64_t mask = same_digit(digit, bits, active);
      const int first = active ? __ffsll((unsigned long long)mask) - 1 : lane;
      int old = 0;
      if (active && lane == first) old = atomicAdd(&counters[digit], __popcll(mask));
      place[b] = __shfl(old, first, 64) + __popcll(mask & ((1ull << lane) - 1));
    }
  }
  __device__ __forceinline__ void scatter(int shift, int bits, const int* begins, const SortOut& out) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int b = 0; b < kSortItems; ++b)
      if (b * 64 + lane < count) out.write(begins[(pair[b].x >> shift) & ((1u << bits) - 1)] + place[b], pair[b]);
  }
};

template <int THREADS>
__device__ __forceinline__ void sort_zero(SortLds<THREADS>& l) {
  for (int i = threadIdx.x; i < l.kWaves * kSortBins; i += THREADS) (&l.counters[0][0])[i] = 0;
  __syncthreads();
}

// Exclusive sum over the workgroup's threads.
template <int THREADS>
__device__ __forceinline__ int sort_scan(int v, SortLds<THREADS>& l) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = v;
  for (int i = 1; i < 64; i <<= 1) {
    const int o = __shfl_up(s, i, 64);
    if (lane >= i) s += o;
  }
  __syncthreads();
  if (lane == 63) l.scan[w] = s;
  __syncthreads();
  int base = 0;
  for (int i = 0; i < w; ++i) base += l.scan[i];
  return base + s - v;
}

// The tile's count of the thread's digit (0: the thread has none).
template <int THREADS>
__device__ __forceinline__ int sort_digit_count(const SortLds<THREADS>& l) {
  int sum = 0;
  if (threadIdx.x < kSortBins) {
#pragma unroll
    for (int w = 0; w < l.kWaves; ++w) sum += l.counters[w][threadIdx.x];
  }
  return sum;
}

// Turns the waves' counts into the places where their digits begin, given where
// the tile's digits begin (one digit per thread).
template <int THREADS>
__device__ __forceinline__ void sort_places(SortLds<THREADS>& l, int begin) {
  if (threadIdx.x < kSortBins) {
#pragma unroll
    for (int w = 0; w < l.kWaves; ++w) {
      const int c = l.counters[w][threadIdx.x];
      l.counters[w][threadIdx.x] = begin;
      begin += c;
    }
  }
  __syncthreads();
}

// Marks every token's run as empty, a part by each workgroup.
__device__ __forceinline__ void clear_bounds(int2* bounds, int vocab, int block, int blocks) {
  for (int v = block * blockDim.x + threadIdx.x; v < vocab; v += blocks * blockDim.x) bounds[v] = make_int2(0, 0);
}

// counts[tile][digit]; bounds (or null) is cleared on the way.
__global__ __launch_bounds__(kSortThreads) void k_sort_count(SortSource src, SortShape s, int shift, int bits,
                                                             int* counts, int2* bounds) {
  __shared__ SortLds<kSortThreads> l;
  SortChunk chunk;
  chunk.load(src, s, blockIdx.x);
  if (bounds) clear_bounds(bounds, s.vocab, blockIdx.x, gridDim.x);
  sort_zero(l);
  chunk.rank(shift, bits, l.counters[threadIdx.x >> 6]);
  __syncthreads();
  counts[blockIdx.x * kSortBins + threadIdx.x] = sort_digit_count(l);
}

// For more than kSortTiles tiles: counts[t] becomes the sum of the tiles before
// t, counts[tiles] the sum of all.  A workgroup per 64 digits, a wave per eighth
// of the tiles.
__global__ __launch_bounds__(kSortThreads) void k_sort_prefix(int* counts, int tiles) {
  __shared__ int sums[kSortWaves][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, digit = blockIdx.x * 64 + lane;
  const int each = (tiles + kSortWaves - 1) / kSortWaves;
  const int from = w * each < tiles ? w * each : tiles, to = from + each < tiles ? from + each : tiles;
  int sum = 0;
#pragma unroll 16
  for (int t = from; t < to; ++t) sum += counts[t * kSortBins + digit];
  sums[w][lane] = sum;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < w; ++i) before += sums[i][lane];
#pragma unroll 16
  for (int t = from; t < to; ++t) {
    const int c = counts[t * kSortBins + digit];
    counts[t * kSortBins + digit] = before;
    before += c;
  }
  if (w == kSortWaves - 1) counts[tiles * kSortBins + digit] = before;
}

__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(SortSource src, SortShape s, int shift, int bits,
                                                               const int* counts, SortOut out) {
  __shared__ SortLds<kSortThreads> l;
  SortChunk chunk;
  chunk.load(src, s, blockIdx.x);
  int before = 0, total = 0;
  if (s.tiles > kSortTiles) {
    before = counts[blockIdx.x * kSortBins + threadIdx.x];
    total = counts[s.tiles * kSortBins + threadIdx.x];
  } else {
#pragma unroll 32
    for (int t = 0; t < s.tiles; ++t) {
      const int c = counts[t * kSortBins + threadIdx.x];
      total += c;
      before += t < (int)blockIdx.x ? c : 0;
    }
  }
  sort_zero(l);
  int* mine = l.counters[threadIdx.x >> 6];
  chunk.rank(shift, bits, mine);
  const int begin = sort_scan(total, l) + before;
  sort_places(l, begin);
  chunk.scatter(shift, bits, mine, out);
}

// All passes by the first workgroup (n <= kSortOne, one tile); the others clear
// the bounds.
__global__ __launch_bounds__(kSortOneThreads) void k_sort_one(Tokens tokens, SortShape s, int passes, int bits,
                                                           uint2* even, uint2* odd, SortOut last, int2* bounds) {
  __shared__ SortLds<kSortOneThreads> l;
  if (blockIdx.x > 0) {
    clear_bounds(bounds, s.vocab, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  int* mine = l.counters[threadIdx.x >> 6];
  for (int pass = 0; pass < passes; ++pass) {
    const SortSource src{tokens, pass == 0 ? nullptr : pass & 1 ? even : odd};
    const SortOut out = pass == passes - 1 ? last : SortOut{pass & 1 ? odd : even, nullptr, nullptr};
    SortChunk chunk;
    chunk.load(src, s, 0);
    sort_zero(l);
    chunk.rank(pass * bits, bits, mine);
    __syncthreads();
    const int begin = sort_scan(sort_digit_count(l), l);
    sort_places(l, begin);
    chunk.scatter(pass * bits, bits, mine, out);
    __syncthreads();
  }
}

// ---- sums of runs ----
//
// Pieces: 32 sorted positions, and blocks of 8 pieces, each at a multiple of its
// size.  A piece (block) of one token alone is summed on its own, so that a
// token that fills half the batch is summed by as many waves as any others.

constexpr int kPiece = 32, kBlockPieces = 8, kBlock = kPiece * kBlockPieces;

// Sums of rows, added in order: a lane's vector in each of NC stretches of 64 N
// columns.
template <class T, int NC>
struct RowSum {
  static constexpr int N = Vec<T>::N;
  float acc[NC][N];
  int at[NC], n[NC];  // the lane's vectors (vec_begin)
  __device__ __forceinline__ RowSum(int col, int d) {
#pragma unroll
    for (int c = 0; c < NC; ++c) at[c] = vec_begin<N>(col + c * 64 * N, d, n[c]);
    zero();
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[c][e] = 0.f;
  }
  // rows of `src`, row(i) for i in [0, count)
  template <class S, int U, class F>
  __device__ __forceinline__ void add(const S* src, int count, F row) {
    constexpr int M = Vec<S>::N, P = N / M;  // vectors of S per stretch and lane
    int i = 0;
    for (; i + U <= count; i += U) {
      typename Vec<S>::raw v[U][NC][P];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const S* p = src + row(i + u);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int q = 0; q < P; ++q) v[u][c][q] = load_raw(p + at[c] + q * M, n[c] - q * M);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int q = 0; q < P; ++q) {
            float f[M];
            Vec<S>::unpack(v[u][c][q], f);
#pragma unroll
            for (int e = 0; e < M; ++e) acc[c][q * M + e] += f[e];
          }
    }
    for (; i < count; ++i) {
      const S* p = src + row(i);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int q = 0; q < P; ++q) {
          float v[M];
          load_row(p + at[c] + q * M, n[c] - q * M, v);
#pragma unroll
          for (int e = 0; e < M; ++e) acc[c][q * M + e] += v[e];
        }
    }
  }
};

struct Runs {
  const int* keys;       // sorted
  const int* positions;
  int64_t n;
  int vocab;
  int2* bounds;          // of each token's run: first and last + 1; 0, 0 for none
};

// One workgroup of 8 waves per block of 256 positions, each wave a piece:
// piece_sums[piece] for a piece of one token, block_sums[block] if the whole
// block is of one (then no piece_sums).  The first column's workgroups also note
// where the runs begin and end.  Small pieces, so that a few frequent tokens are
// spread over all CUs: 524288 tokens, 1024 bf16 features 115 us, 78848 tokens, 768
// features 16 us (pieces of 64 in blocks of 1024: 190 and 46).
template <class T>
__global__ __launch_bounds__(kBlockPieces * 64) void k_embed_pieces(Runs runs, const T* dy, int64_t lddy, int d,
                                                                    float* piece_sums, float* block_sums) {
  constexpr int N = Vec<T>::N;
  __shared__ float lds[kBlockPieces][64 * N];
  const int64_t b0 = (int64_t)blockIdx.x * kBlock;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t p0 = b0 + w * kPiece, at = p0 + lane;
  // the wave's keys, and the one before and after
  const bool in = lane < kPiece && at < runs.n;
  const int key = in ? runs.keys[at] : runs.vocab;
  const int pos = in ? runs.positions[at] : 0;
  const int last = b0 + kBlock <= runs.n ? runs.keys[b0 + kBlock - 1] : runs.vocab;
  const int first = runs.keys[b0];
  if (blockIdx.y == 0 && in && key < runs.vocab) {
    if (at == 0 || runs.keys[at - 1] != key) runs.bounds[key].x = (int)at;
    if (at + 1 == runs.n || runs.keys[at + 1] != key) runs.bounds[key].y = (int)at + 1;
  }
  const bool all = first == last && first < runs.vocab;
  const int key0 = __builtin_amdgcn_readlane(key, 0);
  const bool one = key0 < runs.vocab && key0 == __builtin_amdgcn_readlane(key, kPiece - 1);
  if (!__syncthreads_or(one)) return;
  const int col = blockIdx.y * 64 * N + lane * N;
  RowSum<T, 1> sum(col, d);
  if (one)
    sum.template add<T, 16>(dy, kPiece, [&](int i) { return (int64_t)__builtin_amdgcn_readlane(pos, i) * lddy; });
  if (!all) {
    if (one) {
#pragma unroll
      for (int q = 0; q < N / 4; ++q) {
        const float v[4] = {sum.acc[0][q * 4], sum.acc[0][q * 4 + 1], sum.acc[0][q * 4 + 2], sum.acc[0][q * 4 + 3]};
        store_row(piece_sums + (p0 / kPiece) * d + sum.at[0] + q * 4, sum.n[0] - q * 4, v);
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e) lds[w][e * 64 + lane] = sum.acc[0][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * N; i += kBlockPieces * 64) {
    int n;
    const int c = vec_begin<N>(blockIdx.y * 64 * N + (i & 63) * N, d, n);
    float s = 0.f;
    for (int p = 0; p < kBlockPieces; ++p) s += lds[p][i];
    if ((i >> 6) < n) block_sums[(int64_t)blockIdx.x * d + c + (i >> 6)] = s;
  }
}

constexpr int kWaveRows = 4, kDwRows = 4 * kWaveRows;  // vocabulary rows per wave, per workgroup
// Up to here nothing is sorted: every workgroup picks the positions of its own rows
// out of all tokens.  One launch instead of three, and on autograd's thread a launch takes
// longer than that (one token alone is 512 rows by four waves).
constexpr int kFew = 512;

// The positions of a workgroup's kDwRows rows among kFew tokens at most, in order.
struct FewTokens {
  Tokens tokens;
  int64_t padding;
};
struct FewLds {
  int positions[kFew];
  int counts[4][kDwRows];
};
// Fills l.positions, and gives lane r < kDwRows of every wave the bounds of row r's.
__device__ __forceinline__ int2 few_positions(const FewTokens& few, int n, int v0, int vocab, FewLds& l) {
  constexpr int kPer = kFew / 256;  // tokens per lane
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (threadIdx.x < 4 * kDwRows) (&l.counts[0][0])[threadIdx.x] = 0;
  __syncthreads();
  int row[kPer], place[kPer];
  uint64_t mask[kPer];
#pragma unroll
  for (int b = 0; b < kPer; ++b) {
    const int i = w * (kFew / 4) + b * 64 + lane;
    const int64_t tok = i < n ? few.tokens[i] : -1, r = tok - v0;
    const bool mine = tok >= 0 && tok < vocab && tok != few.padding && r >= 0 && r < kDwRows;
    row[b] = mine ? (int)r : -1;
    mask[b] = same_digit(mine ? (uint32_t)r : 0u, 4, mine);
    const int first = mine ? __ffsll((unsigned long long)mask[b]) - 1 : lane;
    int old = 0;
    if (mine && lane == first) old = atomicAdd(&l.counts[w][row[b]], __popcll(mask[b]));
    place[b] = __shfl(old, first, 64) + __popcll(mask[b] & ((1ull << lane) - 1));
  }
  __syncthreads();
  int total = 0, before = 0;
  if (lane < kDwRows) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      total += l.counts[q][lane];
      before += q < w ? l.counts[q][lane] : 0;
    }
  }
  int end = total;
  for (int i = 1; i < kDwRows; i <<= 1) {
    const int o = __shfl_up(end, i, 64);
    if (lane >= i) end += o;
  }
  const int begin = end - total;
#pragma unroll
  for (int b = 0; b < kPer; ++b) {
    const int at = __shfl(begin + before, row[b] < 0 ? 0 : row[b], 64) + place[b];
    if (row[b] >= 0) l.positions[at] = w * (kFew / 4) + b * 64 + lane;
  }
  __syncthreads();
  return lane < kDwRows ? make_int2(begin, end) : make_int2(0, 0);
}

constexpr int kShortRun = 16;  // a wave's work alone; longer ones would be the launch's last

// Bound by memory and, for few tokens, by the latency of positions, then rows of dy:
// dW of 131072 x 1024 bf16 in 144 us, of 49408 x 768 in 32 us, of 32001 x 641 fp32 in 18.
// Every row of dW, four to a wave: the positions of their runs of up to 16 are
// one list, whose rows of dy are loaded one after another across the ends of the
// runs.  Longer runs are summed by the workgroup's 4 waves together, with the
// pieces' sums.
template <class T, int NC, bool PAST>
__global__ __launch_bounds__(256) void k_embed_rows(Runs runs, FewTokens few, const T* dy, int64_t lddy, int d,
                                                    float scale, const float* piece_sums, const float* block_sums,
                                                    T* dw) {
  constexpr int N = Vec<T>::N;
  constexpr int U = 8 / NC;      // rows of dy in flight
  constexpr int UF = U > 1 ? U / 2 : 1;  // rows of sums
  __shared__ float lds[3][NC * N * 64];
  __shared__ FewLds few_lds;
  const int v0 = blockIdx.x * kDwRows;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = blockIdx.y * NC * 64 * N + lane * N;
  int2 bound = make_int2(0, 0);
  if (!runs.bounds)
    bound = few_positions(few, (int)runs.n, v0, runs.vocab, few_lds);
  else if (lane < kDwRows && v0 + lane < runs.vocab)
    bound = runs.bounds[v0 + lane];
  auto position = [&](int64_t i) { return runs.bounds ? runs.positions[i] : few_lds.positions[i]; };
  RowSum<T, NC> sum(col, d);
  auto write = [&](int v) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum.acc[c][e] = scaled(scale, sum.acc[c][e]);
      store_row<PAST>(dw + (int64_t)v * d + sum.at[c], sum.n[c], sum.acc[c]);
    }
    sum.zero();
  };
  // the wave's short runs as one list
  int begin[kWaveRows], end[kWaveRows + 1];  // of the run; of its part of the list
  end[0] = 0;
#pragma unroll
  for (int r = 0; r < kWaveRows; ++r) {
    const int q = w * kWaveRows + r;
    begin[r] = __builtin_amdgcn_readlane(bound.x, q);
    const int count = __builtin_amdgcn_readlane(bound.y, q) - begin[r];
    end[r + 1] = end[r] + (count <= kShortRun ? count : 0);
    if (count == 0 && v0 + q < runs.vocab) write(v0 + q);
  }
  const int total = end[kWaveRows];
  int r = 0;
  for (int i0 = 0; i0 < total; i0 += 64) {
    const int i = i0 + lane;
    int at = begin[0];
#pragma unroll
    for (int k = 1; k < kWaveRows; ++k) at = i >= end[k] ? begin[k] - end[k] : at;
    const int pos = i < total ? position(at + i) : 0;
    const int n = total - i0 < 64 ? total - i0 : 64;
    for (int j = 0; j < n; j += U) {
      typename Vec<T>::raw v[U][NC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const T* p = dy + (int64_t)__builtin_amdgcn_readlane(pos, j + u < n ? j + u : n - 1) * lddy;
#pragma unroll
        for (int c = 0; c < NC; ++c) v[u][c] = load_raw(p + sum.at[c], sum.n[c]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j + u >= n) break;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float f[N];
          Vec<T>::unpack(v[u][c], f);
#pragma unroll
          for (int e = 0; e < N; ++e) sum.acc[c][e] += f[e];
        }
        // (the list's runs are not empty but for those that were written above or are long)
        const int done = i0 + j + u + 1;
#pragma unroll
        for (int k = 0; k < kWaveRows; ++k)
          if (done == end[k + 1] && end[k] < done) write(v0 + w * kWaveRows + k);
      }
    }
  }
  const uint64_t longer = __ballot(bound.y - bound.x > kShortRun);
  for (uint64_t left = longer; left; left &= left - 1) {
    const int q = __ffsll((unsigned long long)left) - 1;
    const int64_t lo = __builtin_amdgcn_readlane(bound.x, q), hi = __builtin_amdgcn_readlane(bound.y, q);
    // [lo, a) positions, [a, a2) pieces, [a2, b2) blocks, [b2, b) pieces, [b, hi) positions
    int64_t a = (lo + kPiece - 1) / kPiece * kPiece, b = hi / kPiece * kPiece;
    if (a > b || !runs.bounds) a = b = hi;
    int64_t a2 = (a + kBlock - 1) / kBlock * kBlock, b2 = b / kBlock * kBlock;
    if (a2 >= b2) a2 = b2 = b;
    sum.zero();
    auto positions = [&](int64_t from, int64_t to) {  // a quarter for each wave
      const int count = (int)(to - from), each = (count + 3) / 4;
      const int end = (w + 1) * each < count ? (w + 1) * each : count;
      for (int at = w * each; at < end; at += 64) {
        const int mine = end - at < 64 ? end - at : 64;
        const int pos = lane < mine ? position(from + at + lane) : 0;
        sum.template add<T, U>(dy, mine, [&](int i) { return (int64_t)__builtin_amdgcn_readlane(pos, i) * lddy; });
      }
    };
    auto sums = [&](const float* s, int64_t from, int64_t to) {
      const int64_t count = to - from, each = (count + 3) / 4;
      const int64_t at = w * each < count ? w * each : count;
      const int mine = (int)(count - at < each ? count - at : each);
      sum.template add<float, UF>(s, mine, [&](int i) { return (from + at + i) * (int64_t)d; });
    };
    positions(lo, a);
    sums(piece_sums, a / kPiece, a2 / kPiece);
    sums(block_sums, a2 / kBlock, b2 / kBlock);
    sums(piece_sums, b2 / kPiece, b / kPiece);
    positions(b, hi);
    __syncthreads();
    if (w > 0) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < N; ++e) lds[w - 1][(c * N + e) * 64 + lane] = sum.acc[c][e];
    }
    __syncthreads();
    if (w == 0) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < N; ++e)
          for (int p = 0; p < 3; ++p) sum.acc[c][e] += lds[p][(c * N + e) * 64 + lane];
      write(v0 + q);
    }
  }
}

}  // namespace mec
