// Attention on the MFMA cores: what its forward and backward kernels share.
//
//   s_ij = scale q_i . k_j,  p_ij = exp(s_ij) / sum over the keys that i sees,
//   o_i = sum_j p_ij v_j
// and for a gradient do of o, with delta_i = do_i . o_i,
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i.
// No matrix of scores is kept: the forward leaves one number a row,
// lse_i = log2 sum_j exp(s_ij), from which the backward makes p_ij anew.
//
// Tiles.  A wave works on 32 rows of its own ("columns" of the MFMA's result,
// one a lane: lanes l and l + 32 share one) against blocks of 32 rows of a tile
// in LDS.  v_mfma_f32_32x32x16 leaves a lane 16 of the 32 block rows,
// 8 (i / 4) + 4 (l / 32) + i % 4 in register i.  As the next product sums over
// just these rows, in any order that both operands share, registers 8 s .. 8 s + 7
// rounded to 16 bits are its right operand as they stand, and its left operand,
// the other tile transposed, is read from LDS in that order by
// ds_read_b64_tr_b16: probabilities never leave their lane.  fp32 runs the same
// kernels on v_mfma_f32_32x32x2, eight to a step of 16.
//
// LDS holds a tile as rows of VPR 16-byte vectors, vector v of row r in place
// v ^ swz(r): 16 rows at one vector (row reads) lie in 16 different groups of 4
// banks, and so do 4 rows by 4 vectors (transposed reads).
#pragma once
#include "mec_vec.h"

namespace mec {
namespace attn {

constexpr uint32_t OOB = 0x80000000u;  // buffer offset that reads as zero
constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char Lds;

using View = HeadsView;

struct Problem {
  View q, k, v, g;  // g: the gradient of the result
  int queries, keys, heads, key_heads, group, d;
  int64_t pairs;    // batch * key_heads
  int causal;
  float scale, c;   // c = scale log2(e)
  const void *query_lengths, *key_lengths;
  int length64;
  // number of queries and keys of batch entry b, each within what there is
  __device__ __forceinline__ int length(const void* p, int64_t b, int all) const {
    if (p == nullptr) return all;
    const int64_t n = length64 ? ((const int64_t*)p)[b] : (int64_t)((const int32_t*)p)[b];
    return __builtin_amdgcn_readfirstlane(n < 0 ? 0 : n > all ? all : (int)n);  // (the same in all lanes: scalar)
  }
  __device__ __forceinline__ int nq(int64_t b) const { return length(query_lengths, b, queries); }
  __device__ __forceinline__ int nk(int64_t b) const { return length(key_lengths, b, keys); }
};

// What the workgroups of a launch take: `tiles` items of each pair of batch entry and
// key head.  Workgroups run on the 8 XCDs in turn, each with an L2 of its own.  With many
// pairs an XCD has all items of its pairs, one pair after another, which share what they
// read.  With few pairs the first items of all pairs come first (where causal, the
// longest), and an XCD has a pair's items in turn with others: in the order of many
// pairs some XCDs would have all the long items, the others all the short ones.
struct Items {
  int64_t count, ids;  // of items; the same, as a multiple of 8
  static constexpr int MANY = 64;
  __device__ __forceinline__ bool take(int64_t pairs, int tiles, int64_t& pair, int& tile) const {
    int64_t id = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (id >= ids) return false;
    if (pairs >= MANY) {
      id = (id & 7) * (ids >> 3) + (id >> 3);
      pair = id / tiles;
      tile = (int)(id - pair * tiles);
    } else {
      tile = (int)(id / pairs);
      pair = id - tile * pairs;
    }
    return id < count;
  }
};

// 8 consecutive k of a row or column, and the products of 32 x 16 by 16 x 32.
template <class T>
struct Ops {
  static constexpr bool F32 = std::is_same<T, float>::value, F16 = std::is_same<T, _Float16>::value;
  struct Frag32 {
    float v[8];
  };
  using Frag = typename std::conditional<F32, Frag32, i16x8>::type;
  static constexpr int EPV = 16 / sizeof(T);
  // fp16 probabilities are kept 2^6 times as large: beside a row's largest (1 to 2^8,
  // as the running maximum may lag by 8) those down to 2^-30 are not flushed
  static constexpr float BIAS = F16 ? 6.f : 0.f;
  // in the backward, where they are at most 1, 2^14 times
  static constexpr float GRAD_BIAS = F16 ? 14.f : 0.f, GRAD_UNIT = F16 ? 0x1p-14f : 1.f;

  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) c = mfma_f32_32x32x2(a.v[e], b.v[e], c);
      return c;
    } else {
      return mfma16_32x32x16<F16>(a, b, c);
    }
  }
  // registers 8 s .. 8 s + 7 as a right operand, rounded to T
  static __device__ __forceinline__ Frag pack(const f32x16& x, int s) {
    Frag f;
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f.v[e] = x[8 * s + e];
    } else {
      u32x4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = F16 ? pack2_f16(x[8 * s + 2 * e], x[8 * s + 2 * e + 1]) : pack2_bf16(x[8 * s + 2 * e], x[8 * s + 2 * e + 1]);
      f = __builtin_bit_cast(i16x8, r);
    }
    return f;
  }
  // sum + the 8 values of a fragment
  static __device__ __forceinline__ float add(const Frag& f, float sum) {
    if constexpr (!F32) {
      const uint32_t ones = F16 ? 0x3c003c00u : 0x3f803f80u;
      const u32x4 r = __builtin_bit_cast(u32x4, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (F16)
          sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, (uint32_t)r[e]), __builtin_bit_cast(f16x2, ones), sum, false);
        else
          sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, (uint32_t)r[e]), __builtin_bit_cast(bf16x2, ones),
                                                sum, false);
      }
    }
    return sum;
  }
  // k 16 s + 8 half .. + 7 of a row of d elements in memory
  static __device__ __forceinline__ Frag load_row(const T* row, bool valid, int s, int half, int d) {
    const int at = 16 * s + 8 * half, n = valid ? d - at : 0;
    Frag f;
    if constexpr (F32) {
      const auto lo = load_raw(row + at, n), hi = load_raw(row + at + 4, n - 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f.v[e] = __uint_as_float(lo[e]);
        f.v[4 + e] = __uint_as_float(hi[e]);
      }
    } else {
      f = __builtin_bit_cast(i16x8, (u32x4)load_raw(row + at, n));
    }
    return f;
  }
  static __device__ __forceinline__ float dot(const Frag& a, const Frag& b) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (F32)
        sum += a.v[e] * b.v[e];
      else if constexpr (F16)
        sum += (float)__builtin_bit_cast(f16x8, a)[e] * (float)__builtin_bit_cast(f16x8, b)[e];
      else
        sum += bf16_to_f32((uint16_t)a[e]) * bf16_to_f32((uint16_t)b[e]);
    }
    return sum;
  }
};

// A tile of rows of 32 DB elements in LDS.
template <class T, int DB>
struct Tile {
  using O = Ops<T>;
  using Frag = typename O::Frag;
  static constexpr int EPV = O::EPV, VPR = 32 * DB / EPV, RB = 16 * VPR;
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (VPR % 16 == 0)
      return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (VPR % 16 == 8)
      return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else
      return (r >> 2) & 3;
  }
  // A lane's part of the addresses below.  Of 16-bit rows all of them are two numbers, xor and plus constants (a row's
  // beginning is a multiple of the xored bits): held as such they take 2 registers, where the compiler keeps up to 16
  // (see `again`).
  static constexpr bool XOR = !O::F32;
  static constexpr int STEPS = VPR % 16 == 0 ? 7 : VPR % 16 == 8 ? 3 : 1;  // the bits of a step that are xored
  struct At {
    int lane, row, col;
    __device__ __forceinline__ explicit At(int l) : lane(l), row(0), col(0) {
      if constexpr (XOR) {
        const int r = l & 31, half = l >> 5, j = l & 15;
        row = r * RB + ((half ^ swz(r)) << 4);
        const int w = 2 * ((l >> 4) & 1) + ((j & 3) >> 1), high = swz(j >> 2) & ~3;
        col = (4 * half + (j >> 2)) * RB + ((high | (w ^ half)) << 4) + 8 * (j & 1);
      }
    }
    // from here on the addresses are made anew, not kept from before
    __device__ __forceinline__ void again() {
      if constexpr (XOR) asm volatile("" : "+v"(row), "+v"(col));
    }
  };
  static __device__ __forceinline__ Frag row(Lds* tile, int row0, int s, const At& at) {
    if constexpr (XOR)
      return *(__attribute__((address_space(3))) i16x8*)(tile + row0 * RB + (at.row ^ ((s & STEPS) << 5)) +
                                                         ((s & ~STEPS) << 5));
    else
      return row(tile, row0, s, at.lane);
  }
  static __device__ __forceinline__ Frag col(Lds* tile, int row0, int db, const At& at) {
    if constexpr (XOR) {
      typedef __attribute__((address_space(3))) i16x4 Quad;
      // (whole rows of 8 or 16 vectors: the block of 4 vectors is xored, too)
      const int x = STEPS > 1 ? at.col ^ (db << 6) : at.col, plus = STEPS > 1 ? 0 : db << 6;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Quad*)(tile + row0 * RB + x + plus));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Quad*)(tile + (row0 + 8) * RB + (x ^ 32) + plus));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return col(tile, row0, db, at.lane);
    }
  }
  // k 16 s + 8 (lane / 32) .. + 7 of row row0 + lane % 32 (row0 a multiple of 32)
  static __device__ __forceinline__ Frag row(Lds* tile, int row0, int s, int lane) {
    const int r = lane & 31, half = lane >> 5, x = swz(r);
    Lds* at = tile + (row0 + r) * RB;
    if constexpr (O::F32) {
      Frag f;
      const f32x4 lo = *(__attribute__((address_space(3))) f32x4*)(at + (((4 * s + 2 * half) ^ x) << 4));
      const f32x4 hi = *(__attribute__((address_space(3))) f32x4*)(at + (((4 * s + 2 * half + 1) ^ x) << 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f.v[e] = lo[e];
        f.v[4 + e] = hi[e];
      }
      return f;
    } else {
      return *(__attribute__((address_space(3))) i16x8*)(at + (((2 * s + half) ^ x) << 4));
    }
  }
  // (16-bit types) the same, written
  static __device__ __forceinline__ void put_row(Lds* tile, int row0, int s, int lane, const Frag& f) {
    const int r = lane & 31;
    *(__attribute__((address_space(3))) i16x8*)(tile + (row0 + r) * RB + (((2 * s + (lane >> 5)) ^ swz(r)) << 4)) = f;
  }
  // column 32 db + lane % 32, rows row0 + 4 (lane / 32) + {0 .. 3, 8 .. 11} (row0 a multiple of 16)
  static __device__ __forceinline__ Frag col(Lds* tile, int row0, int db, int lane) {
    const int half = lane >> 5;
    if constexpr (O::F32) {
      Frag f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = row0 + 4 * half + 8 * (e >> 2) + (e & 3);
        const int v = (8 * db + ((lane & 31) >> 2)) ^ swz(r);
        f.v[e] = *(__attribute__((address_space(3))) float*)(tile + r * RB + (v << 4) + 4 * (lane & 3));
      }
      return f;
    } else {
      // (lane j of 16 points at 4 columns of row j / 4 and receives column j of 4 rows)
      const int j = lane & 15, v = 4 * db + 2 * ((lane >> 4) & 1) + ((j & 3) >> 1);
      const int r0 = row0 + 4 * half + (j >> 2), r1 = r0 + 8;
      typedef __attribute__((address_space(3))) i16x4 Quad;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Quad*)(tile + r0 * RB + ((v ^ swz(r0)) << 4) + 8 * (j & 1)));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Quad*)(tile + r1 * RB + ((v ^ swz(r1)) << 4) + 8 * (j & 1)));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// ROWS rows of a matrix on their way from memory through the registers of NT
// threads into a tile.
template <class T, int DB, int ROWS, int NT>
struct Loader {
  using Tl = Tile<T, DB>;
  static constexpr int NV = ROWS * Tl::VPR / NT;
  static_assert(NV * NT == ROWS * Tl::VPR, "the vectors divide evenly");
  const char* base;
  int64_t pitch;  // bytes between rows
  int d, t;
  bool whole;     // rows of whole 16-byte vectors on 4-byte boundaries, offsets within a tile in 31 bits
  u32x4 r[NV];

  // (uniform but for t)
  __device__ __forceinline__ void init(const View& v, int64_t b, int h, int d_, int t_) {
    base = (const char*)((const T*)v.p + b * v.batch + (int64_t)h * v.head);
    pitch = v.token * (int64_t)sizeof(T);
    d = d_;
    t = t_;
    whole = d % Tl::EPV == 0 && ((uintptr_t)base & 3) == 0 && (pitch & 3) == 0 && pitch < (int64_t)1 << 24;
  }
  // rows row0 .. row0 + ROWS - 1, those from `valid` rows on as zeros
  __device__ __forceinline__ void load(int row0, int valid) {
    const char* p = base + row0 * pitch;
    if (whole) {
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = t + i * NT, row = at / Tl::VPR, v = at % Tl::VPR;
        const uint32_t off = row < valid && v * Tl::EPV < d ? (uint32_t)(row * (int)pitch + v * 16) : OOB;
        r[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = t + i * NT, row = at / Tl::VPR, v = at % Tl::VPR;
        r[i] = load_raw((const T*)(p + row * pitch) + v * Tl::EPV, row < valid ? d - v * Tl::EPV : 0);
      }
    }
  }
  __device__ __forceinline__ void store(Lds* tile) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = t + i * NT, row = at / Tl::VPR, v = at % Tl::VPR;
      *(__attribute__((address_space(3))) u32x4*)(tile + row * Tl::RB + ((v ^ Tl::swz(row)) << 4)) = r[i];
    }
  }
};

// ROWS rows of a matrix on their way from memory into a tile, past the registers where
// rows are whole 16-byte vectors on 16-byte boundaries.  The loads of a tile are in flight
// while the one before is read: each of the two is an LDS array of its own, which tells the
// compiler that reads of the one need not wait for the other.
template <class T, int DB, int ROWS, int WAVES>
struct Fetcher {
  using Tl = Tile<T, DB>;
  static constexpr int VPR = Tl::VPR, BLOCKS = ROWS * VPR / 64, NB = (BLOCKS + WAVES - 1) / WAVES;
  const char* base;
  int64_t pitch;  // bytes between rows
  int d, lane, wave;
  bool whole;
  uint32_t off[NB];

  // (moves: `move` will be called)
  __device__ __forceinline__ void init(const View& v, int64_t b, int h, int d_, int wave_, int lane_, bool moves = false) {
    base = (const char*)((const T*)v.p + b * v.batch + (int64_t)h * v.head);
    pitch = v.token * (int64_t)sizeof(T);
    d = d_;
    lane = lane_;
    wave = wave_;
    const int64_t apart = moves ? v.head * (int64_t)sizeof(T) : 0;  // a head from the next
    whole = d % Tl::EPV == 0 && (((uintptr_t)base | pitch | apart) & 15) == 0 && pitch < (int64_t)1 << 24;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      // (lane l of the block fills its place l)
      const int at = (i * WAVES + wave) * 64 + lane, row = at / VPR, vec = (at % VPR) ^ Tl::swz(row);
      off[i] = vec * Tl::EPV < d ? (uint32_t)(row * (int)pitch + vec * 16) : OOB;
    }
  }
  // another head of the same matrix (`whole` holds for all of them: see init)
  __device__ __forceinline__ void move(const View& v, int64_t b, int h) {
    base = (const char*)((const T*)v.p + b * v.batch + (int64_t)h * v.head);
  }
  // rows row0 .. row0 + ROWS - 1, those from `valid` rows on as zeros
  __device__ __forceinline__ void load(Lds* tile, int row0, int valid) const {
    const char* p = base + row0 * pitch;
    if (whole) {
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int block = i * WAVES + wave;
        if (BLOCKS % WAVES == 0 || block < BLOCKS) {
          const uint32_t o = valid >= ROWS || (block * 64 + lane) / VPR < valid ? off[i] : OOB;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(tile + block * 1024), 16,
                                                   o, 0, 0, 0);
        }
      }
    } else {
      for (int block = wave; block < BLOCKS; block += WAVES) {
        const int at = block * 64 + lane, row = at / VPR, vec = (at % VPR) ^ Tl::swz(row);
        *(__attribute__((address_space(3))) u32x4*)(tile + at * 16) =
            load_raw((const T*)(p + row * pitch) + vec * Tl::EPV, row < valid ? d - vec * Tl::EPV : 0);
      }
    }
  }
};
// Loads into LDS, and the waves' reads and writes of it, are done for all waves.
__device__ __forceinline__ void loads_done() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): loads that pass no registers too
  __syncthreads();
}
// load(i, 0 or 1) and use(i, 0 or 1) of the tiles first .. last - 1 in two places in turn, the next on its
// way while one is used.  Ends with all uses done.
template <class Load, class Use>
__device__ __forceinline__ void walk_tiles(int first, int last, Load load, Use use) {
  std::integral_constant<int, 0> a;
  std::integral_constant<int, 1> b;
  if (first >= last) return;
  load(first, a);
  loads_done();
#pragma unroll 1
  for (int i = first;;) {
    if (i + 1 < last) load(i + 1, b);
    use(i, a);
    loads_done();
    if (++i >= last) break;
    if (i + 1 < last) load(i + 1, a);
    use(i, b);
    loads_done();
    if (++i >= last) break;
  }
}

// The other half of the wave's value.
__device__ __forceinline__ float other_half(float v) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? sw[0] : sw[1]);
}

// The running maximum m (in units of log2) after scores s, times c: sum l and accumulators o are
// rescaled where it grew by more than 8 in any row.
template <class O, int NB, int DB>
__device__ __forceinline__ void grow(const f32x16 (&s)[NB], float c, float& m, float& l, f32x16 (&o)[DB]) {
  float top = s[0][0];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[b][e]);
  top = fmaxf(top, other_half(top)) * c;
  if (__any(top > m + 8.f)) {
    const float now = fmaxf(m, top), f = now == -kInf ? 1.f : fast_exp2(m - now);
    m = now;
    l *= f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] *= f;
  }
}
template <class O, int DB>
__device__ __forceinline__ void grow(const f32x16& s, float c, float& m, float& l, f32x16 (&o)[DB]) {
  const f32x16 one[1] = {s};
  grow<O>(one, c, m, l, o);
}

// Gradients of scores on their way to fp16 (to the other types they go as they are).  They fall with the number of
// keys, and sums of thousands of them are well within fp16 where each by itself is below its least step, or beyond
// its largest number.  So they are held times a power of two for each row or key (a lane and its other half): it starts
// large, and where one of them would pass 2^15, the row's largest is brought to 2^10 or more; what was summed so far
// follows.  Steps are then at most 2^-34 of the row's largest.  The maximum of a lane's 16 in each block of 32 x 32 costs
// 1 to 5% of a training step in fp16 (256 x 257 tokens, 12 heads of 64: 589 to 613 us; 16384 causal tokens, 16 heads of
// 128 on 4: 5.02 to 5.10 ms).
template <class O>
struct GradUnit {
  float up;
  __device__ __forceinline__ explicit GradUnit(float with = 1.f) : up(O::F16 ? 0x1p46f * with : 1.f) {}
  // (x - y) times the unit, rounded once
  __device__ __forceinline__ float times(float x, float y) const { return O::F16 ? fmaf(x, up, -y * up) : x - y; }
  __device__ __forceinline__ float times(float x) const { return O::F16 ? x * up : x; }
  // a unit's worth
  __device__ __forceinline__ float back() const { return __uint_as_float((254u << 23) - __float_as_uint(up)); }
  // makes ds fit; rescale(f) takes sums of earlier ones times f (where an inf is among ds, all is left as it is)
  template <class Rescale>
  __device__ __forceinline__ void fit(f32x16& ds, Rescale rescale) {
    if constexpr (O::F16) {
      float top = fabsf(ds[0]);
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, fabsf(ds[e]));
      top = fmaxf(top, other_half(top));
      if (__any(top > 0x1p15f)) {
        // 2^10 to 2^11 of the largest, by the exponents
        const float f = top > 0x1p15f && top < kInf ? __uint_as_float((264u - (__float_as_uint(top) >> 23)) << 23) : 1.f;
        up *= f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] *= f;
        rescale(f);
      }
    }
  }
};
template <int DB>
__device__ __forceinline__ void scale_all(f32x16 (&acc)[DB], float f) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] *= f;
}

// A wave's 32 columns of the accumulators, rounded to T, on their way to rows of d
// elements.  They pass through LDS (32 rows of a tile, of which the wave alone has the
// use), so that 16 bytes a lane and whole lines leave the CU: 8 bytes a lane, 32 rows at
// a time, are four times the requests, which short sequences wait for.
template <class T, int DB>
struct Rows {
  using Tl = Tile<T, DB>;
  typedef typename std::conditional<sizeof(T) == 4, float, uint32_t>::type E;
  typedef E Four __attribute__((ext_vector_type(sizeof(T))));  // 4 elements
  Four v[DB][4];

  __device__ __forceinline__ void pack(const f32x16 (&acc)[DB], float f) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = acc[db][4 * i] * f, b = acc[db][4 * i + 1] * f, c = acc[db][4 * i + 2] * f,
                    d = acc[db][4 * i + 3] * f;
        if constexpr (sizeof(T) == 4)
          v[db][i] = Four{a, b, c, d};
        else if constexpr (std::is_same<T, _Float16>::value)
          v[db][i] = Four{pack2_f16(a, b), pack2_f16(c, d)};
        else
          v[db][i] = Four{pack2_bf16(a, b), pack2_bf16(c, d)};
      }
  }
  __device__ __forceinline__ void put(Lds* mine, int lane) const {
    const int r = lane & 31, half = lane >> 5, x = Tl::swz(r);
    Lds* const to = mine + r * Tl::RB;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4)
          *(__attribute__((address_space(3))) Four*)(to + (((8 * db + 2 * i + half) ^ x) << 4)) = v[db][i];
        else
          *(__attribute__((address_space(3))) Four*)(to + (((4 * db + i) ^ x) << 4) + 8 * half) = v[db][i];
      }
  }
  // row(r): where row r goes, nullptr: nowhere
  template <class Row>
  static __device__ __forceinline__ void flush(Lds* mine, int d, int lane, Row row) {
    constexpr int EPV = Tl::EPV, VPR = Tl::VPR;
    wave_sync();
#pragma unroll
    for (int i = 0; i < VPR / 2; ++i) {
      const int at = i * 64 + lane, r = at / VPR, vec = at % VPR, n = d - vec * EPV;
      T* p = row(r);
      if (p != nullptr && n > 0) {
        const u32x4 x4 = *(__attribute__((address_space(3))) u32x4*)(mine + r * Tl::RB + ((vec ^ Tl::swz(r)) << 4));
        p += vec * EPV;
        if (n >= EPV) {
          *(typename Vec<T>::raw*)p = x4;
        } else {
#pragma unroll
          for (int e = 0; e < EPV - 1; ++e)
            if (e < n) {
              if constexpr (sizeof(T) == 4)
                p[e] = __uint_as_float(x4[e]);
              else
                p[e] = __builtin_bit_cast(T, (uint16_t)(x4[e / 2] >> (16 * (e & 1))));
            }
        }
      }
    }
  }
};
template <class T, int DB, class Row>
__device__ __forceinline__ void store_rows(Lds* mine, const f32x16 (&acc)[DB], float f, int d, int lane, Row row) {
  Rows<T, DB> rows;
  rows.pack(acc, f);
  rows.put(mine, lane);
  Rows<T, DB>::flush(mine, d, lane, row);
}

// 32 rows of LDS for wave 0 .. 3 in the two places of tiles: each holds the rows of two waves, or of all.
template <int STEP, int RB>
__device__ __forceinline__ Lds* wave_rows(char* a, char* b, int wave) {
  return STEP == 64 || wave < 2 ? (Lds*)a + 32 * wave * RB : (Lds*)b + 32 * (wave - 2) * RB;
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

}  // namespace attn
}  // namespace mec
