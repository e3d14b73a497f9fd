// Attention of prompts in float16.
#include "bw_prompt.h"

int bw_launch_prompt_f16(const PromptArgs& a, uint32_t grid, int groups, hipStream_t stream) {
    return with_head<BW_F16>(a.dim, [&](auto head) { return groups == 1 ? launch_prompt<decltype(head), 1>(a, grid, stream) : launch_prompt<decltype(head), 2>(a, grid, stream); });
}
