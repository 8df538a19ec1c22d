// Attention's backward for fp32.
#include "mec_attn_launch.h"

template void mec::attn::launch_backward<float>(const Launch&);
