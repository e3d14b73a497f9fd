"""cache_attention where the weights of the softmax show: values that cancel."""
import pytest
import torch

from attention_ref import Batch, half_step

pytestmark = pytest.mark.gpu


def _filled(b):
    b.cache.write(b.k, b.v, torch.cat(b.slots))
    return b


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_cancel(dtype):
    """Weights of a few tokens that are nearly the same and values 1 and -1: what comes out is the difference of float32 weights.  A score is one product
    (exact in float32); scaling, exponent, exponential, sums and the quotient are at most 16 float32 operations on a weight and one for every token."""
    lengths = [2, 3, 4, 5, 6, 7, 8] * 20
    b = Batch(lengths, 16, 4, 64, 16, 16, 64, dtype, seed=5)
    b.k[..., 1:] = 0
    b.k[..., 0] = torch.rand(b.k.shape[:2], device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(dtype)
    b.v = torch.where(b.v > 0.5, 1.0, -1.0).to(dtype)
    _filled(b)
    out = b.attend()
    at = 0
    worst = 0.0
    for s, n in enumerate(lengths):
        k, v = b.k[at:at + n].double(), b.v[at:at + n].double()
        at += n
        scores = b.q[s].double()[:, 0].view(4, 4, 1) * k[..., 0].t()[:, None] * 64 ** -0.5
        want = torch.matmul(torch.softmax(scores, -1), v.transpose(0, 1).contiguous()).view(16, 64)
        bound = half_step(dtype) * want.abs() + (16 + n) * 2.0 ** -24 + 2.0 ** -25
        worst = max(worst, ((out[s].double() - want).abs() / bound).max().item())
    assert worst <= 1, f"{worst:.3f} times the bound"
