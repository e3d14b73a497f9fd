// The attention kernel over 4-bit codes.
#include "bw_attention.h"

void bw_launch_attention_w4(const AttentionArgs& a, int group, uint32_t grid, hipStream_t stream) { launch_codes<4>(a, group, grid, stream); }
