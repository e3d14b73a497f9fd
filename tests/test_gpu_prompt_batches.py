"""prompt_attention over as many short sequences as the forward takes: its gradients, which have more workgroups than one launch."""
import pytest
import torch

import bitween_amd as bw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,tokens,heads,dim", [(131072, 1, 64, 8), (150000, 2, 63, 8)])
def test_many_short_sequences_are_what_they_are_in_smaller_batches(sequences, tokens, heads, dim):
    """Over 2^23 workgroups of each of the gradients' kernels; every sequence has the bits that it has among a few thousand."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, grad = (torch.randn(sequences, tokens, heads, dim, device="cuda", generator=gen, dtype=torch.float16) for _ in range(4))

    def run(at):
        leaves = [t[at].detach().requires_grad_(True) for t in (q, k, v)]
        out = bw.prompt_attention(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, grad[at])]

    got = run(slice(None))
    if tokens == 1:                                              # one weight, of 1
        assert torch.equal(got[0], v) and torch.equal(got[3], grad)
    for first in range(0, sequences, 10000):
        at = slice(first, first + 10000)
        assert all(torch.equal(a[at], b) for a, b in zip(got, run(at))), first


def test_keys_of_sequences_without_rows():
    """No new token at all, in more sequences than one launch has workgroups: zeros."""
    starts = torch.zeros(2 ** 18 + 1, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(300, 64, 8, device="cuda", dtype=torch.float16, requires_grad=True) for _ in range(2))
    q = torch.zeros(0, 64, 8, device="cuda", dtype=torch.float16, requires_grad=True)
    out = bw.prompt_attention(q, k, v, starts, starts)
    dk, dv = torch.autograd.grad(out, (k, v), torch.zeros_like(out))
    assert out.shape == q.shape and not dk.any() and not dv.any()
