// Scaled token embedding: y_t = scale W[tok_t], and its gradient
// dW_v = scale sum_{t: tok_t = v} dy_t.
#pragma once
#include "mec_vocab.h"

namespace mec {

// The product in 32 bits, then rounded: not contracted into one instruction that
// rounds the exact product to 16 bits.
template <class T>
__device__ __forceinline__ void put_scaled(T* p, float scale, float v) {
#pragma clang fp contract(off)
  float s = scale * v;
  asm("" : "+v"(s));
  put(p, s);
}

// One workgroup per token.  A token outside [0, vocab) gives a row of NaN.
template <class T>
__global__ __launch_bounds__(256) void k_embed(Tokens tokens, const T* weight, int64_t ldw, int64_t vocab, int d,
                                               float scale, T* out) {
  const int64_t t = blockIdx.x, tok = tokens[t];
  const bool ok = tok >= 0 && tok < vocab;
  for (int j = threadIdx.x; j < d; j += 256)
    put_scaled(out + t * d + j, scale, ok ? value(weight[tok * ldw + j]) : NAN);
}

// One workgroup per vocabulary row and 256 features: it looks through all
// tokens and adds the rows of dy of its own, in order.
template <class T>
__global__ __launch_bounds__(256) void k_embed_grad(Tokens tokens, int64_t rows, const T* dy, int64_t lddy, int d,
                                                    float scale, int64_t padding, T* dw) {
  __shared__ int hits[256];
  __shared__ int wave_hits[4];
  const int64_t v = blockIdx.x;
  const int j = blockIdx.y * 256 + threadIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float s = 0.f;
  if (v != padding)
    for (int64_t t0 = 0; t0 < rows; t0 += 256) {
      const int64_t t = t0 + threadIdx.x;
      const bool hit = t < rows && tokens[t] == v;
      const uint64_t mask = __ballot(hit);
      if (lane == 0) wave_hits[w] = __popcll(mask);
      if (!__syncthreads_or(hit)) continue;
      int at = __popcll(mask & ((1ull << lane) - 1)), n = 0;
      for (int i = 0; i < 4; ++i) at += i < w ? wave_hits[i] : 0, n += wave_hits[i];
      if (hit) hits[at] = threadIdx.x;
      __syncthreads();
      if (j < d)
        for (int i = 0; i < n; ++i) s += value(dy[(t0 + hits[i]) * lddy + j]);
      __syncthreads();
    }
  if (j < d) put_scaled(dw + v * d + j, scale, s);
}

}  // namespace mec
