// Host checks shared by the operators of a tower's attention.
#pragma once
#include <type_traits>

#include "mec_host.h"

namespace mec {

constexpr int64_t kMaxHeadsStride = int64_t(1) << 40;

// f(pointer to float, bf16 bits or fp16) for dtype
template <class F>
void with_element_type(int dtype, F f) {
  if (dtype == MEC_DTYPE_F32)
    f((float*)nullptr);
  else if (dtype == MEC_DTYPE_BF16)
    f((uint16_t*)nullptr);
  else
    f((_Float16*)nullptr);
}

inline int check_element_type(int dtype) {
  if (dtype != MEC_DTYPE_F32 && dtype != MEC_DTYPE_BF16 && dtype != MEC_DTYPE_F16)
    return fail(MEC_ERR_INVALID, "dtype %d is not MEC_DTYPE_F32, _BF16 or _F16", dtype);
  return MEC_OK;
}

inline int check_heads(const mec_heads_t* h, const char* what) {
  if (h == nullptr || h->data == nullptr) return fail(MEC_ERR_INVALID, "%s must be non-null", what);
  for (int64_t s : {h->batch_stride, h->token_stride, h->head_stride})
    if (s < 0 || s > kMaxHeadsStride)
      return fail(MEC_ERR_INVALID, "%s: stride %lld out of range [0, 2^40]", what, (long long)s);
  return MEC_OK;
}

inline int check_scratch(const void* workspace, int64_t bytes, int64_t need) {
  if (need > 0 && workspace == nullptr) return fail(MEC_ERR_INVALID, "workspace must be non-null");
  if (bytes < need)
    return fail(MEC_ERR_INVALID, "workspace of %lld bytes, %lld needed", (long long)bytes, (long long)need);
  if (((uintptr_t)workspace & 15) != 0) return fail(MEC_ERR_INVALID, "workspace must be 16-byte aligned");
  return MEC_OK;
}

}  // namespace mec
