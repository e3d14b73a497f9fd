// bw_attention.h - launches of the attention kernel over codes (bw_attention_w8.hip, bw_attention_w4.hip), as bw_attention.hip calls them.
#pragma once
#include "bw_attention_kernel.h"

void bw_launch_attention_w8(const AttentionArgs& a, int group, uint32_t grid, hipStream_t stream);
void bw_launch_attention_w4(const AttentionArgs& a, int group, uint32_t grid, hipStream_t stream);

// One kernel for every number of groups that a head of up to 256 values has, and for up to 4, 8 and 16 queries of a segment.
template <int BITS, int GROUPS, int GS> static void launch_codes(const AttentionArgs& a, uint32_t grid, hipStream_t stream) {
    if (a.dim == GROUPS * GS) {
        if (a.queries <= 4) launch_attention<FormatQ<BITS, GROUPS, GS>, 4>(a, grid, stream);
        else if (a.queries <= 8) launch_attention<FormatQ<BITS, GROUPS, GS>, 2>(a, grid, stream);
        else launch_attention<FormatQ<BITS, GROUPS, GS>, 1>(a, grid, stream);
    } else if constexpr (GROUPS > 1) {
        launch_codes<BITS, GROUPS - 1, GS>(a, grid, stream);
    }
}
template <int BITS> static void launch_codes(const AttentionArgs& a, int group, uint32_t grid, hipStream_t stream) {
    if (group == 32) launch_codes<BITS, 8, 32>(a, grid, stream);
    else if (group == 64) launch_codes<BITS, 4, 64>(a, grid, stream);
    else launch_codes<BITS, 2, 128>(a, grid, stream);
}
