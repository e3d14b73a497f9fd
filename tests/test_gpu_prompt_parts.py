"""prompt_attention where the keys of a row are cut into parts that a second kernel joins: tokens with nothing to see, infinities and NaN, the keys' gradient."""
import pytest
import torch

import bitween_amd as bw
from bitween_amd.kernels import hip_loader
from attention_ref import half_step
from prompt_ref import close, visible
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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk,dim", [(1, 700, 128), (4, 1500, 64), (63, 2063, 128), (9, 2000, 256)])
def test_the_outputs_rounding_is_not_in_the_keys_gradient(nq, nk, dim, dtype):
    """Values of multiples of 1/16 within 2 of 8 (exact in both types), so that the output and its rounding are large beside what the keys' gradient is made of.  Bounds of every value, h
    being half a step:

    dS = P (dP - delta), of which the products take h of itself; P errs by loose = 2 (dim + 16) 2^-24 of the scores' magnitudes + 2 n 2^-24; dP by (dim + 2) 2^-23 of |g| |v|; delta in float32 by
    dim 2^-23 of |g out| and n 2^-23 of sum |dS|, and with what the output errs by (`off`: h |out| + (h + loose) P |v|) only by that part of it by which the weights do not add up to 1, h + loose.
    dK = scale sum dS q: these, n 2^-23 of |dS| |q|, and its own rounding."""
    h, small, scale = half_step(dtype), 2.0 ** -37 if dtype == torch.float16 else 0.0, dim ** -0.5
    gen = torch.Generator(device="cuda").manual_seed(nk + dim)
    q, g = (torch.randn(nq, 2, dim, device="cuda", generator=gen).to(dtype) for _ in range(2))
    k = torch.randn(nk, 2, dim, device="cuda", generator=gen).to(dtype)
    v = (8 + torch.randint(-32, 33, (nk, 2, dim), device="cuda", generator=gen) / 16).to(dtype)
    assert _is_cut(q, k)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dk = torch.autograd.grad(bw.prompt_attention(*leaves), leaves, g)[1]
    seen = visible(nq, nk, None, 0)
    for n in range(2):
        x, y, z, up = (t.detach()[:, n].double() for t in (q, k, v, g))
        p = (x @ y.t() * scale).masked_fill(~seen, float("-inf")).softmax(-1)
        out, dp = p @ z, up @ z.t()
        delta = (up * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        loose = 2 * (dim + 16) * 2.0 ** -24 * (x.abs() @ y.abs().t() * scale * seen).amax(-1, keepdim=True) + 2 * nk * 2.0 ** -24
        off = h * out.abs() + (h + loose) * (p @ z.abs()) + small * (seen.double() @ z.abs()) + 2.0 ** -25
        of_delta = (up.abs() * off).sum(-1, keepdim=True)
        wrong = h * ds.abs() + p * (loose * (dp - delta).abs() + (dim + 2) * 2.0 ** -23 * (up.abs() @ z.abs().t()) + dim * 2.0 ** -23 * (up * out).abs().sum(-1, keepdim=True)
                                    + (h + loose) * of_delta + nk * 2.0 ** -23 * ds.abs().sum(-1, keepdim=True)) + small * ds.abs().amax(0, keepdim=True)
        want = scale * (ds.t() @ x)
        bound = scale * ((wrong * seen).t() @ x.abs() + nk * 2.0 ** -23 * (ds.abs().t() @ x.abs())) + h * want.abs() + 2.0 ** -25
        close(dk[:, n], want, bound, "dk")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk,heads,kv,dim", [(63, 2063, 4, 1, 128), (512, 512, 4, 2, 128), (9, 2000, 2, 2, 256)])
def test_each_gradient_alone(nq, nk, heads, kv, dim, dtype):
    q, k, v, grad = _inputs(nq, nk, heads, kv, dim, dtype, seed=5)
    full = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(bw.prompt_attention(*full), full, grad)
    for wanted in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        some = [t.detach().clone().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(bw.prompt_attention(*some), [some[i] for i in wanted], grad)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, wanted)), wanted
