"""What the weights that prompt_attention's gradients compute again may be off by, over rows of few keys."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import half_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,keys,dim", [(8192, 3, 64), (8192, 6, 64), (4096, 6, 96), (4096, 12, 128), (2048, 6, 256), (1, 700, 128)])
def test_one_row_over_few_keys(batch, keys, dim, dtype):
    """dV = P g of one row.  P is 2^(S c - lse), and lse is log2 of the sum of the forward's weights as they were rounded, each off by h of itself at most (h being half a step), and so their sum
    by h of itself, and all of P with it.  Beside that P is rounded once (h of itself), and so is the result; a score errs by (dim + 16) 2^-24 of its products' magnitudes, itself and in
    the sum by which it is divided, and sums over n keys by n 2^-24 (twice)."""
    h, small, scale = half_step(dtype), 2.0 ** -36 if dtype == torch.float16 else 0.0, dim ** -0.5
    gen = torch.Generator(device="cuda").manual_seed(keys + dim)
    q, g = (torch.randn(batch, 1, 2, dim, device="cuda", generator=gen).to(dtype) for _ in range(2))
    k, v = ((0.5 * torch.randn(batch, keys, 2, dim, device="cuda", generator=gen)).to(dtype) for _ in range(2))
    alone = v.clone().requires_grad_(True)
    (only,) = torch.autograd.grad(bw.prompt_attention(q, k, alone), [alone], g)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dv = torch.autograd.grad(bw.prompt_attention(*leaves), leaves, g)[2]
    assert torch.equal(only, dv)
    x, y, up = (t.detach().double() for t in (q, k, g))
    p = ((x * y).sum(-1) * scale).softmax(1)[..., None]         # [batch, keys, heads, 1]
    loose = 2 * (dim + 16) * 2.0 ** -24 * ((x.abs() * y.abs()).sum(-1) * scale).amax(1, keepdim=True)[..., None] + 2 * keys * 2.0 ** -24
    want = p * up
    bound = (2 * h + loose) * want.abs() + small * up.abs()
    bound = bound * (1 + h) + h * want.abs() + 2.0 ** -25
    worst = ((dv.double() - want).abs() / bound).max().item()
    assert worst <= 1, worst
