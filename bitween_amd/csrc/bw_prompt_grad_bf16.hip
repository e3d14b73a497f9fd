// Gradients of the attention of prompts in bfloat16.
#include "bw_prompt_grad.h"

int bw_launch_prompt_grad_bf16(const PromptGradArgs& g, const PromptGrids& grids, hipStream_t stream) {
    return with_head<BW_BF16>(g.p.dim, [&](auto head) { return launch_prompt_grad<decltype(head)>(g, grids, stream); });
}
