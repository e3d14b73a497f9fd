// bw_prompt_grad.h - launches of the gradients of the prompt attention by type (bw_prompt_grad_f16.hip, bw_prompt_grad_bf16.hip), as bw_prompt_grad.hip calls them.
#pragma once
#include "bw_prompt.h"
#include "bw_prompt_grad_kernel.h"

// Workgroups of each kernel (0: not launched) and what is theirs alone of the arguments: tiles and parts.
struct PromptGrids { uint32_t rows, row_tiles, keys, key_tiles, key_splits, far, far_combos; };

int bw_launch_prompt_grad_f16(const PromptGradArgs& g, const PromptGrids& grids, hipStream_t stream);
int bw_launch_prompt_grad_bf16(const PromptGradArgs& g, const PromptGrids& grids, hipStream_t stream);

template <class H> static int launch_prompt_grad(PromptGradArgs g, const PromptGrids& grids, hipStream_t stream) {
    static uint64_t done[3] = {};
    const void* kernels[3] = {(const void*)prompt_query_grad_kernel<H>, (const void*)prompt_key_grad_kernel<H, true>, (const void*)prompt_key_grad_kernel<H, false>};
    for (int i = 0; i < 3; i++)
        if (!bw_allow_big_lds(kernels[i], done[i])) return BW_ELAUNCH;
    constexpr int kKeyStages = 2 * (2 * H::kTileBytes + 512);
    if (grids.rows) {
        g.p.tiles = grids.row_tiles;
        g.p.splits = 1;
        hipLaunchKernelGGL(prompt_query_grad_kernel<H>, dim3(grids.rows), dim3(256), 4 * H::kTileBytes, stream, g);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    if (grids.far) {
        PromptGradArgs f = g;
        f.p.combos = grids.far_combos;
        f.p.by_combos = FastDiv(grids.far_combos);
        hipLaunchKernelGGL((prompt_key_grad_kernel<H, true>), dim3(grids.far), dim3(256), kKeyStages, stream, f);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    if (grids.keys) {
        g.p.tiles = grids.key_tiles;
        g.p.splits = (int)grids.key_splits;
        hipLaunchKernelGGL((prompt_key_grad_kernel<H, false>), dim3(grids.keys), dim3(256), kKeyStages, stream, g);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}
