"""What is left of a row's dS, which add up to zero, does not meet what all its keys have in common, nor the output's rounding the keys' gradient."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import half_step

pytestmark = pytest.mark.gpu


def _check(seed, batch, tokens, window, dim, dtype):
    """Keys of multiples of 1/16 within 2 of 8 (exact in both types).  Bounds of every value, h being half a step:

    out errs by `off` = h |out| + (h + loose) P |v|, loose = 2 (dim + 16) 2^-24 of the scores' magnitudes + 2 n 2^-24 (see prompt_ref), P by loose of itself.
    dS = P (dP - delta): h of itself, P's error, (dim + 2) 2^-23 of |g| |v| for dP, and delta's.  dQ's delta comes with the rounded output: sum |g| off.  dK's is that of P: of it only the part by which the weights
    do not add up to 1 (h + loose) is left, and sums of n terms in float32.
    dQ = scale sum dS (K - c), c the mean of the last 32 keys that the row sees, whose weights are rounded (h of |c|): dS's errors meet K - c, their sum h |c|; float32 sums n 2^-23 of |dS| |K|."""
    h = half_step(dtype)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q, v, g = (torch.randn(batch, tokens, 2, dim, device="cuda", generator=gen).to(dtype) for _ in range(3))
    k = (8 + torch.randint(-32, 33, (batch, tokens, 2, dim), device="cuda", generator=gen) / 16).to(dtype)
    small = 2.0 ** -37 if dtype == torch.float16 else 0.0
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(bw.prompt_attention(*leaves, window=window), leaves, g)
    q, k, v, g, dq, dk = (t.detach().double().transpose(1, 2).flatten(0, 1) for t in (q, k, v, g, dq, dk))          # [batch x heads, tokens, dim]
    scale, at = dim ** -0.5, torch.arange(tokens, device="cuda")
    seen = (at[None] <= at[:, None]) & (at[None] > at[:, None] - (window or tokens))
    p = torch.matmul(q, k.transpose(1, 2).contiguous()).mul(scale).masked_fill(~seen, float("-inf")).softmax(-1)
    out, dp = torch.matmul(p, v), torch.matmul(g, v.transpose(1, 2).contiguous())
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    reach = (torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()) * scale * seen).amax(-1, keepdim=True)
    loose = 2 * (dim + 16) * 2.0 ** -24 * reach + 2 * tokens * 2.0 ** -24
    off = h * out.abs() + (h + loose) * torch.matmul(p, v.abs()) + small * torch.matmul(seen.double().expand_as(p), v.abs()) + 2.0 ** -25
    of_delta = (g.abs() * off).sum(-1, keepdim=True)
    common = h * ds.abs() + p * (loose * (dp - delta).abs() + (dim + 2) * 2.0 ** -23 * torch.matmul(g.abs(), v.abs().transpose(1, 2).contiguous()) + dim * 2.0 ** -23 * (g * out).abs().sum(-1, keepdim=True))
    for_q = (common + p * of_delta + small * ds.abs().amax(-1, keepdim=True)) * seen
    for_k = (common + p * ((h + loose) * of_delta + tokens * 2.0 ** -23 * ds.abs().sum(-1, keepdim=True)) + small * ds.abs().amax(-2, keepdim=True)) * seen
    mean = seen & (at[None] > at[:, None] - 32)
    c = torch.matmul(mean.double() / mean.sum(-1, keepdim=True), k)
    want_q, want_k = scale * torch.matmul(ds, k), scale * torch.matmul(ds.transpose(1, 2).contiguous(), q)
    apart = (for_q[..., None] * (k[:, None] - c[:, :, None]).abs()).sum(2)
    bound_q = scale * (apart + h * for_q.sum(-1, keepdim=True) * c.abs() + tokens * 2.0 ** -23 * torch.matmul(ds.abs(), k.abs())) + h * want_q.abs() + 2.0 ** -25
    bound_k = scale * (torch.matmul(for_k.transpose(1, 2).contiguous(), q.abs()) + tokens * 2.0 ** -23 * torch.matmul(ds.abs().transpose(1, 2).contiguous(), q.abs())) + h * want_k.abs() + 2.0 ** -25
    return ((dq - want_q).abs() / bound_q).max().item(), ((dk - want_k).abs() / bound_k).max().item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,window,dim", [(2, None, 64), (3, None, 128), (5, None, 128), (5, 2, 256), (40, 6, 128), (70, None, 64)])
def test_what_all_keys_share_is_not_in_the_gradient(tokens, window, dim, dtype):
    of_q, of_k = _check(tokens + dim, 64, tokens, window, dim, dtype)
    assert of_q <= 1 and of_k <= 1, (of_q, of_k)
