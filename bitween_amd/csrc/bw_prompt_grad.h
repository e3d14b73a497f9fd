// bw_prompt_grad.h - launches of the gradients of the prompt attention by type (bw_prompt_grad_f16.hip, bw_prompt_grad_bf16.hip), as bw_prompt.hip calls them.
#pragma once
#include "bw_prompt.h"
#include "bw_prompt_grad_kernel.h"

// Workgroups of each kernel (0: not launched), tiles of each sequence where they are not listed, and joins at most.
struct PromptGrids { uint32_t rows, row_tiles, keys, key_tiles, joins; };

int bw_launch_prompt_grad_f16(const PromptGradArgs& g, const PromptGrids& grids, hipStream_t stream);
int bw_launch_prompt_grad_bf16(const PromptGradArgs& g, const PromptGrids& grids, hipStream_t stream);

// Workgroups of 256 threads in several launches where they would pass the 2^32 threads of one; `before`: of those in the launches before.
constexpr uint32_t kLaunchBlocks = 1u << 23;
template <class F> static int in_launches(uint32_t blocks, uint32_t& before, F&& launch) {
    for (before = 0; before < blocks; before += kLaunchBlocks) {
        launch(dim3(blocks - before < kLaunchBlocks ? blocks - before : kLaunchBlocks));
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}

template <class H> static int launch_prompt_grad(PromptGradArgs g, const PromptGrids& grids, hipStream_t stream) {
    static uint64_t done[2] = {};
    const void* kernels[2] = {(const void*)prompt_query_grad_kernel<H>, (const void*)prompt_key_grad_kernel<H>};
    for (int i = 0; i < 2; i++)
        if (!bw_allow_big_lds(kernels[i], done[i])) return BW_ELAUNCH;
    if (grids.rows) {
        g.p.set_tiles(grids.row_tiles);
        if (int st = in_launches(grids.rows + (g.plan ? 1 : 0), g.before, [&](dim3 grid) { hipLaunchKernelGGL(prompt_query_grad_kernel<H>, grid, dim3(256), 4 * H::kTileBytes, stream, g); }))
            return st;
        if (g.p.splits > 1) {
            const int threads = g.p.dim / 4;
            const uint32_t rows = (uint32_t)(g.p.q_tokens * g.p.q_heads), per = 256 / threads;
            hipLaunchKernelGGL(prompt_query_join_kernel<H::kType>, dim3((rows + per - 1) / per), dim3(256), 0, stream, g, threads, rows);
            if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
            g.p.set_splits(1);
        }
    }
    if (!grids.keys) return BW_OK;
    g.p.set_tiles(grids.key_tiles);
    if (int st = in_launches(grids.keys, g.before, [&](dim3 grid) { hipLaunchKernelGGL(prompt_key_grad_kernel<H>, grid, dim3(256), 2 * kKeyStage<H>, stream, g); })) return st;
    if (grids.joins) {
        const int chunks = (kGradKeys * 2 * g.p.dim + 1023) / 1024;
        hipLaunchKernelGGL(prompt_grad_join_kernel<H::kType>, dim3(grids.joins * g.p.kv_heads * chunks), dim3(256), 0, stream, g, chunks);
        if (hipGetLastError() != hipSuccess) return BW_ELAUNCH;
    }
    return BW_OK;
}
