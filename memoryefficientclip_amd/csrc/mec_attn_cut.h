// Attention's backward: how its work is cut, and its launches for one element type.
#pragma once
#include "mec_attn_host.h"

namespace mec {
namespace attn {

// Waves and LDS of k_attn_whole_grad, 0 waves where it does not fit.  Where it does it is the faster form at all sizes
// (a step's time less the forward's, 256 x 12 heads, us, this form and two kernels that walk over tiles; bf16, heads of 64:
// 77 tokens 135 and 138, 129 205 and 307, 197 306 and 398, 257 442 and 630; 1024 x 77 causal 230 and 580; heads of 32:
// 77 tokens 140 and 146, 257 270 and 320; of 72: 77 tokens 128 and 173, 160 277 and 393; fp32, 77 tokens of 64, 391 and 467).
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
