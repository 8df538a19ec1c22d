// Attention's backward for fp16.
#include "mec_attn_launch.h"

template void mec::attn::launch_backward<_Float16>(const Launch&);
