"""prompt_attention where there are many workgroups, whose keys are neither cut into parts nor shared by groups of waves: against 64 bits."""
import pytest
import torch

import bitween_amd as bw
from prompt_ref import close, reference
from test_gpu_prompt import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads,kv,dim,window,sinks", [(1601, 32, 8, 128, None, 0), (1601, 32, 8, 128, 300, 70), (1700, 24, 24, 64, None, 0), (1333, 32, 16, 96, 500, 1), (1100, 60, 60, 80, None, 0)])
def test_one_sequence(tokens, heads, kv, dim, window, sinks, dtype):
    q, k, v, grad = _inputs(tokens, tokens, heads, kv, dim, dtype, seed=tokens + dim)
    _check(q, k, v, grad, [(0, tokens, 0, tokens)], (), window, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_heads_of_256(dtype):
    q, k, v, grad = _inputs(1200, 1200, 64, 64, 256, dtype, seed=1)
    _check(q, k, v, grad, [(0, 1200, 0, 1200)], (), None, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 3)])
def test_packed_sequences(window, sinks, dtype):
    cuts = [0, 700, 701, 701, 1900, 2500]
    q, k, v, grad = _inputs(2500, 2500, 32, 8, 128, dtype, seed=3)
    starts = torch.tensor(cuts, device="cuda", dtype=torch.int32)
    _check(q, k, v, grad, [(a, b, a, b) for a, b in zip(cuts, cuts[1:])], (starts,), window, sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads", [(1600, 32), (200, 2)])
def test_infinities_and_nan_touch_what_sees_them(tokens, heads, dtype):
    """One value that is not finite, one key and head: outputs and gradients beside its channel, its rows and its head are as without it, bit for bit."""
    q, k, v, grad = _inputs(tokens, tokens, heads, heads, 128, dtype, seed=4)
    window, at = 100, tokens // 2

    def run(value):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        with torch.no_grad():
            leaves[2][at, 1, 5] = value
        out = bw.prompt_attention(*leaves, window=window)
        return [out.detach(), *torch.autograd.grad(out, leaves, grad)]

    want = run(0.0)
    for bad in (float("inf"), float("nan")):
        out, dq, dk, dv = run(bad)
        sees = torch.zeros(tokens, dtype=torch.bool, device="cuda")
        sees[at:at + window] = True
        assert not torch.isfinite(out[sees, 1, 5]).any()
        beside = torch.ones_like(out, dtype=torch.bool)
        beside[sees, 1, 5] = False
        assert torch.equal(out[beside], want[0][beside])
        assert torch.equal(dq[~sees], want[1][~sees]) and torch.equal(dq[:, 0], want[1][:, 0]) and torch.isfinite(dq[~sees]).all()
        far = torch.ones(tokens, dtype=torch.bool, device="cuda")
        far[at - window + 1:at + window] = False                 # keys that no row shares with it
        assert torch.equal(dk[far], want[2][far]) and torch.equal(dv[far], want[3][far])


def test_rows_are_what_they_are_alone():
    """The same rows with their sequence alone and among many: the cut of the work differs, the results by their roundings only."""
    q, k, v, _ = _inputs(1500, 1500, 32, 8, 128, torch.bfloat16, seed=6)
    all_heads = bw.prompt_attention(q, k, v)
    want = reference(q[:, :4], k[:, :1], v[:, :1], [(0, 1500, 0, 1500)], None, 0, 128 ** -0.5)[0]
    close(all_heads[:, :4], *want, "many")
    close(bw.prompt_attention(q[:, :4], k[:, :1], v[:, :1]), *want, "few")
