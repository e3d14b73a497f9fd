"""prompt_attention where the keys of a row are cut into parts that a second kernel joins."""
import pytest
import torch

import bitween_amd as bw
from bitween_amd.kernels import hip_loader
from prompt_ref import visible
from test_gpu_prompt import _check, _inputs

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _is_cut(q, k, starts=(), window=None, sinks=0):
    at = [t.data_ptr() for t in starts] or [None, None]
    p = hip_loader.Prompt(q.shape[0], k.shape[0], *at, len(starts[0]) - 1 if starts else 1, q.shape[1], k.shape[1], q.shape[2], window or 0, sinks, 0.1)
    return hip_loader.load().bw_prompt_attention_workspace_bytes(p) > 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk,heads,kv,dim", [(1100, 1000, 1, 1, 128), (1100, 1024, 1, 1, 64), (2100, 2048, 4, 2, 128), (600, 512, 2, 1, 256)])
def test_more_queries_than_keys(nq, nk, heads, kv, dim, dtype):
    q, k, v, grad = _inputs(nq, nk, heads, kv, dim, dtype, seed=nq)
    assert _is_cut(q, k)
    out = bw.prompt_attention(q, k, v)
    assert not out[:nq - nk].any(), "tokens with nothing to see are zeros"
    _check(q, k, v, grad, [(0, nq, 0, nk)], (), None, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1500, 3)])
@pytest.mark.parametrize("news,alls,heads,kv,dim", [([10, 40, 200, 50], [3, 1700, 190, 107], 2, 2, 64), ([20, 5, 15], [0, 1990, 10], 4, 2, 128)])
def test_more_queries_than_keys_in_one_of_the_sequences(news, alls, heads, kv, dim, window, sinks, dtype):
    starts = [torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32) for n in (news, alls)]
    q, k, v, grad = _inputs(sum(news), sum(alls), heads, kv, dim, dtype, seed=dim)
    assert _is_cut(q, k, starts, window, sinks)
    at = [s.tolist() for s in starts]
    _check(q, k, v, grad, [(at[0][s], at[0][s + 1], at[1][s], at[1][s + 1]) for s in range(len(news))], starts, window, sinks)


def test_a_row_without_a_finite_score_is_not_an_empty_one():
    """A row whose only scores are minus infinity gives NaN where keys are in parts too; one that sees no key zeros."""
    q, k, v, _ = _inputs(1100, 1000, 1, 1, 128, torch.float16)
    q, k = q.abs().contiguous(), k.clone()
    k[0, 0, 0] = float("-inf")
    out = bw.prompt_attention(q, k, v)
    assert not out[:100].any() and torch.isnan(out[100]).all() and torch.isfinite(out[101:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk,heads,kv,dim,window,sinks", [(512, 512, 4, 2, 128, None, 0), (1024, 1024, 8, 2, 128, None, 0), (63, 2063, 4, 1, 128, None, 0), (600, 512, 2, 1, 256, None, 0),
                                                             (130, 1500, 2, 1, 96, None, 0), (200, 8000, 2, 1, 64, 4000, 3)])
def test_infinities_and_nan_touch_what_sees_them(nq, nk, heads, kv, dim, window, sinks, dtype):
    """One value of q, k, v or the gradient is an infinity or a NaN: what does not see its token (or is not seen by it) has the bits that it has without."""
    base = [t.contiguous() for t in _inputs(nq, nk, heads, kv, dim, dtype, seed=4)]

    def run(q, k, v, grad):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = bw.prompt_attention(*leaves, window=window, sinks=sinks)
        return [out.detach(), *torch.autograd.grad(out, leaves, grad)]

    clean = run(*base)
    seen = visible(nq, nk, window, sinks)
    for which in range(4):
        n = base[which].shape[0]
        for token, value in ((n - 1, float("inf")), (n - 7, float("nan")), (n - 20, float("-inf")), (n - 45, float("inf")), (n // 2, float("nan")), (3, float("-inf"))):
            t = [x.clone() for x in base]
            t[which][token, -1, 5] = value
            got = run(*t)
            if which in (1, 2):
                rows = seen[:, token]
                keys = seen[rows].any(0)
            else:
                rows = torch.zeros(nq, dtype=torch.bool, device="cuda")
                rows[token] = True
                keys = seen[token]
            for name, g, c, touched in zip(("out", "dq", "dk", "dv"), got, clean, (rows, rows, keys, keys)):
                assert torch.equal(g[~touched], c[~touched]), (name, which, token, value)
            if which == 2:
                assert not torch.isfinite(got[0][rows][:, -1, 5]).any()
            if which == 1:
                assert not torch.isfinite(got[1][rows][:, -1, 5]).any()
