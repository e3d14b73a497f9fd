// The attention kernel over 8-bit codes.
#include "bw_attention.h"

void bw_launch_attention_w8(const AttentionArgs& a, int group, uint32_t grid, hipStream_t stream) { launch_codes<8>(a, group, grid, stream); }
