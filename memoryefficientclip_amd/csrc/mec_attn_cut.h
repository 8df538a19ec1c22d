// Attention's backward: how its work is cut, and its launches for one element type.
#pragma once
#include "mec_attn_host.h"

namespace mec {
namespace attn {

// Waves and LDS of k_attn_whole_grad, 0 waves where it does not fit.  Where it does it was the faster form at all
// sizes, 2 to 256 x 12 heads (256 x 12 heads of 64, us, this form and two kernels that walk over tiles: 77 tokens 68
// and 131, 197 tokens 297 and 354, 257 tokens 414 and 571; fp32, 77 tokens, 395 and 459).
struct Whole {
  int waves;
  size_t lds;
};

// How the work of the two kernels that walk over tiles is cut.
struct Cut {
  bool few_rows, few_keys;  // 32 of them a workgroup, not 128
  int row_tiles, key_tiles, splits;
  int64_t delta, parts;     // bytes
};

// (each element type has a source of its own: they compile side by side)
struct Launch {
  Problem a;
  Whole whole;
  Cut cut;
  Grid gq, gk, gj;
  const float* lse;
  float *delta, *parts;
  const void* out;
  void *dq, *dk, *dv;
  hipStream_t stream;
};
template <class T>
void launch_backward(const Launch& l);

}  // namespace attn
}  // namespace mec
