// Rows of fp32, bf16 or fp16 elements in 16-byte vectors, at any alignment and
// with any number of elements, as fp32 values.
#pragma once
#include "mec_common.h"

namespace mec {

__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float value(_Float16 v) { return (float)v; }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = f32_to_bf16(v); }
__device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }

// 16 bytes in memory at the alignment of a 2- or 4-byte element.
template <int ALIGN>
struct Bytes16;
template <>
struct Bytes16<2> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Bytes16<4> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};

// 16 bytes of elements at any alignment, as floats.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  using raw = typename Bytes16<sizeof(T)>::type;
  static __device__ __forceinline__ void unpack(const raw& r, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, float>::value) {
        v[i] = __uint_as_float(r[i]);
      } else if constexpr (std::is_same<T, uint16_t>::value) {
        v[2 * i] = __uint_as_float(r[i] << 16);
        v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
      } else {
        const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)r[i]);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      }
    }
  }
  static __device__ __forceinline__ raw pack(const float (&v)[N]) {
    raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, float>::value)
        r[i] = __float_as_uint(v[i]);
      else if constexpr (std::is_same<T, uint16_t>::value)
        r[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
      else
        r[i] = pack2_f16(v[2 * i], v[2 * i + 1]);
    }
    return r;
  }
};

// p[i] for i < n (n may be <= 0), zero bits beyond.
template <class T>
__device__ __forceinline__ typename Vec<T>::raw load_raw(const T* p, int n) {
  constexpr int N = Vec<T>::N;
  if (n >= N) return *(const typename Vec<T>::raw*)p;
  typename Vec<T>::raw r = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) {
      if constexpr (sizeof(T) == 4)
        r[i] = __float_as_uint(p[i]);
      else
        r[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (16 * (i & 1));
    }
  return r;
}
template <class T>
__device__ __forceinline__ void load_row(const T* p, int n, float (&v)[Vec<T>::N]) {
  Vec<T>::unpack(load_raw(p, n), v);
}

// Outputs that pass half of the last-level cache (256 MB) are stored past it: there
// they would only push out what is read next, and their lines hold up the kernel
// that follows while they are written back.  Smaller ones stay for their reader.
// (PAST is a template argument: the compiler joins the two stores of a branch into
// one without the hint.)
constexpr int64_t kKeepBytes = int64_t(128) << 20;

template <bool PAST, class T>
__device__ __forceinline__ void store_vec(T* p, const typename Vec<T>::raw& v) {
  if constexpr (PAST)
    __builtin_nontemporal_store(v, (typename Vec<T>::raw*)p);
  else
    *(typename Vec<T>::raw*)p = v;
}
template <bool PAST = false, class T>
__device__ __forceinline__ void store_row(T* p, int n, const float (&v)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  if (n >= N) {
    store_vec<PAST>(p, Vec<T>::pack(v));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) put(p + i, v[i]);
  }
}

}  // namespace mec
