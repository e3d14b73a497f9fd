// Attention of prompts in float16.
#include "bw_prompt.h"

int bw_launch_prompt_f16(const PromptArgs& a, uint32_t grid, hipStream_t stream) {
    return with_head<BW_F16>(a.dim, [&](auto head) { return launch_prompt<decltype(head)>(a, grid, stream); });
}
