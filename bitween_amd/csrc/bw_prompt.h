// bw_prompt.h - launches of the prompt attention's kernels by type (bw_prompt_f16.hip, bw_prompt_bf16.hip), as bw_prompt.hip calls them.
#pragma once
#include "bw_prompt_kernel.h"

int bw_launch_prompt_f16(const PromptArgs& a, uint32_t grid, int groups, hipStream_t stream);
int bw_launch_prompt_bf16(const PromptArgs& a, uint32_t grid, int groups, hipStream_t stream);

// f(Head) for the smallest head that holds `dim` values.
template <int DT, class F> static int with_head(int dim, F&& f) {
    if (dim <= 64) return f(Head<DT, 64>{});
    if (dim <= 96) return f(Head<DT, 96>{});
    if (dim <= 128) return f(Head<DT, 128>{});
    return f(Head<DT, 256>{});
}

template <class H, int GROUPS> static int launch_prompt(const PromptArgs& a, uint32_t grid, hipStream_t stream) {
    static uint64_t done = 0;
    if (!bw_allow_big_lds((const void*)prompt_forward_kernel<H, GROUPS>, done)) return BW_ELAUNCH;
    hipLaunchKernelGGL((prompt_forward_kernel<H, GROUPS>), dim3(grid), dim3(256), 4 * H::kTileBytes * GROUPS, stream, a);
    return hipGetLastError() == hipSuccess ? BW_OK : BW_ELAUNCH;
}
