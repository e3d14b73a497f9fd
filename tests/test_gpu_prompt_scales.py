"""prompt_attention with scales that are nothing or next to it, over scores near the end of float32."""
import pytest
import torch

import bitween_amd as bw
from prompt_ref import close, reference
from test_gpu_prompt import _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -140, -(2.0 ** -145)])
@pytest.mark.parametrize("nq,nk", [(150, 150), (3, 2000)])
def test_scores_that_are_scaled_away_weigh_the_same(nq, nk, scale):
    """Queries and keys of 2^60: scores up to 2^127, which a scale of 0 leaves at 0, and one of 2^-140 at 2^-13 at most."""
    q, k, v, grad = _inputs(nq, nk, 4, 2, 64, torch.bfloat16, seed=8)
    q, k = (t.clamp(-3, 3) * 2.0 ** 59 for t in (q, k))
    assert 2.0 ** 118 < torch.matmul(q[:, 0].float(), k[:, 0].float().t()).abs().max() < 2.0 ** 127
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = bw.prompt_attention(*leaves, scale=scale)
    got = [out.detach(), *torch.autograd.grad(out, leaves, grad)]
    want = reference(q, k, v, [(0, nq, 0, nk)], None, 0, scale, grad)
    for name, g, (value, bound) in (("out", got[0], want[0]), ("dv", got[3], want[3])):
        close(g, value, bound, name)
    if scale == 0:
        assert not got[1].any() and not got[2].any()
