// Attention's backward for bf16.
#include "mec_attn_launch.h"

template void mec::attn::launch_backward<uint16_t>(const Launch&);
