"""prompt_attention and its gradients against 64 bits, at the sizes, masks and layouts where they can go wrong."""
import pytest
import torch

import bitween_amd as bw
from prompt_ref import close, reference

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _inputs(nq, nk, heads, kv, dim, dtype, seed=0, spread=1.0):
    """Rows of one projection each: queries, and keys and values side by side."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = (spread * torch.randn(nq, heads + 1, dim, device="cuda", generator=gen)).to(dtype)[:, :heads]
    kv_rows = torch.randn(nk, 2 * kv, dim, device="cuda", generator=gen).to(dtype)
    grad = torch.randn(nq, heads, dim, device="cuda", generator=gen).to(dtype)
    return q, kv_rows[:, :kv], kv_rows[:, kv:], grad


def _check(q, k, v, grad, spans, starts, window, sinks, scale=None):
    dim = q.shape[-1]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = bw.prompt_attention(*leaves, *starts, window=window, sinks=sinks, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    plain = bw.prompt_attention(q, k, v, *starts, window=window, sinks=sinks, scale=scale)
    assert torch.equal(plain, out.detach()), "recorded or not"
    got = [out.detach(), *torch.autograd.grad(out, leaves, grad, retain_graph=True)]
    again = torch.autograd.grad(out, leaves, grad)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], again)), "the same inputs give the same bits"
    want = reference(q, k, v, spans, window, sinks, dim ** -0.5 if scale is None else scale, grad)
    for name, g, (value, bound) in zip(("out", "dq", "dk", "dv"), got, want):
        close(g, value, bound, name)


SHAPES = [  # new tokens, tokens, query heads, key heads, dim, window, sinks
    (1, 1, 1, 1, 8, None, 0), (1, 1, 2, 1, 128, 1, 0), (2, 2, 4, 4, 64, None, 0), (1, 300, 8, 2, 128, None, 0), (31, 31, 2, 2, 64, None, 0), (33, 33, 6, 2, 96, 7, 1),
    (64, 64, 4, 1, 128, None, 0), (65, 65, 5, 1, 80, 16, 4), (127, 200, 4, 2, 128, 60, 3), (129, 129, 3, 3, 40, None, 0), (130, 130, 16, 1, 64, 64, 0), (257, 257, 8, 8, 128, 128, 130),
    (300, 300, 2, 1, 256, None, 0), (70, 333, 4, 1, 256, 100, 33), (100, 100, 2, 2, 192, 33, 2), (513, 513, 4, 2, 128, None, 0), (640, 1000, 4, 2, 64, 65, 200), (5, 3, 2, 1, 64, None, 0),
    (200, 70, 4, 2, 128, 16, 2), (90, 90, 2, 1, 120, 1, 0), (90, 90, 2, 1, 64, 1, 1), (64, 64, 7, 7, 72, 64, 64), (1025, 1025, 2, 1, 128, 200, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_one_sequence(shape, dtype):
    nq, nk, heads, kv, dim, window, sinks = shape
    q, k, v, grad = _inputs(nq, nk, heads, kv, dim, dtype)
    _check(q, k, v, grad, [(0, nq, 0, nk)], (), window, sinks)


PACKED = [  # lengths of the sequences' new tokens, of all their tokens, rows in front and behind that belong to none
    ([5, 0, 130, 1, 64], [5, 0, 130, 1, 64], 0, 0), ([1] * 70, [1] * 70, 0, 3), ([40, 3, 0, 200], [40, 90, 17, 333], 7, 9), ([0, 0], [0, 0], 2, 2), ([300], [300], 0, 40),
    ([3] * 200, [3] * 200, 0, 0), ([17, 130], [0, 140], 0, 0), ([128, 128], [128, 128], 128, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (33, 2), (200, 150)])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("packed", range(len(PACKED)))
def test_packed_sequences(packed, heads, kv, dim, window, sinks, dtype):
    news, alls, front, behind = PACKED[packed]
    nq, nk = (front + sum(n) + behind for n in (news, alls))
    q, k, v, grad = _inputs(nq, nk, heads, kv, dim, dtype, seed=packed)
    starts, spans = [], []
    for n in (news, alls):
        starts.append(torch.tensor([front] + n, device="cuda").cumsum(0).to(torch.int32))
    at = [s.tolist() for s in starts]
    spans = [(at[0][s], at[0][s + 1], at[1][s], at[1][s + 1]) for s in range(len(news))]
    # what belongs to no sequence is not looked at
    bad = float("nan")
    q, k, v, grad = q.clone(), k.clone(), v.clone(), grad.clone()
    for t, n in ((q, at[0]), (grad, at[0]), (k, at[1]), (v, at[1])):
        t[:front], t[n[-1]:] = bad, bad
    zero = [torch.nan_to_num(t, nan=0.0) for t in (q, k, v, grad)]
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = bw.prompt_attention(*leaves, starts[0], None if news == alls else starts[1], window=window, sinks=sinks)
    got = [out.detach(), *torch.autograd.grad(out, leaves, grad)]
    want = reference(*zero[:3], spans, window, sinks, dim ** -0.5, zero[3])
    for name, g, (value, bound) in zip(("out", "dq", "dk", "dv"), got, want):
        close(g, value, bound, name)
    for g, n in zip(got, (at[0], at[0], at[1], at[1])):
        assert not g[:front].any() and not g[n[-1]:].any(), "rows of no sequence are zeros"


@pytest.mark.parametrize("dtype", DTYPES)
def test_batches_are_their_sequences(dtype):
    gen = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(3, 100, 4, 64, device="cuda", generator=gen).to(dtype)
    k, v = (torch.randn(3, 170, 2, 64, device="cuda", generator=gen).to(dtype) for _ in range(2))
    grad = torch.randn(3, 100, 4, 64, device="cuda", generator=gen).to(dtype)
    kw = dict(window=50, sinks=3)
    layouts = {"plain": lambda t: t, "heads first": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "odd rows": lambda t: torch.nn.functional.pad(t, (0, 3))[..., :64],
               "off 16 bytes": lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)}
    for name, layout in layouts.items():
        leaves = [layout(t).detach().requires_grad_(True) for t in (q, k, v)]
        out = bw.prompt_attention(*leaves, **kw)
        grads = torch.autograd.grad(out, leaves, layout(grad))
        for b in range(3):
            one = [t[b].detach().requires_grad_(True) for t in (q, k, v)]
            o = bw.prompt_attention(*one, **kw)
            assert torch.equal(o, out[b]), name
            assert all(torch.equal(x, y[b]) for x, y in zip(torch.autograd.grad(o, one, grad[b]), grads)), name
    starts = [torch.arange(4, device="cuda") * n for n in (100, 170)]
    packed = bw.prompt_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), *starts, **kw)
    assert torch.allclose(packed.float(), out.detach().flatten(0, 1).float(), atol=2e-2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_touch_what_sees_them(dtype):
    """One token's row of q, k, v or the gradient is an infinity or a NaN: what does not see it (or is not seen by it) has the bits that it has without."""
    nq, heads, kv, dim, window, sinks = 300, 4, 2, 64, 40, 3
    base = _inputs(nq, nq, heads, kv, dim, dtype, seed=4)
    base = [t.contiguous() for t in base]

    def run(q, k, v, grad):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = bw.prompt_attention(*leaves, window=window, sinks=sinks)
        return [out.detach(), *torch.autograd.grad(out, leaves, grad)]

    clean = run(*base)
    from prompt_ref import visible
    seen = visible(nq, nq, window, sinks)
    for which in range(4):
        for token, value in ((0, float("inf")), (150, float("nan")), (170, float("-inf")), (299, float("inf"))):
            t = [x.clone() for x in base]
            t[which][token, 1, 5] = value
            got = run(*t)
            # rows of q (and out, dq) that meet the token, tokens of k and v that do
            if which in (1, 2):
                rows = seen[:, token]
                keys = seen[rows].any(0)
            else:
                rows = torch.zeros(nq, dtype=torch.bool, device="cuda")
                rows[token] = True
                keys = seen[token]
            for g, c, touched in zip(got, clean, (rows, rows, keys, keys)):
                assert torch.equal(g[~touched], c[~touched]), (which, token, value)
            out_rows = got[0][rows]
            if which == 2:
                assert not torch.isfinite(out_rows[:, 2:, 5]).any() and torch.isfinite(out_rows[:, :2]).all()
            if which == 0:
                assert not torch.isfinite(out_rows[:, 1]).any()


def test_a_score_of_minus_infinity_weighs_nothing():
    q, k, v, grad = _inputs(70, 70, 2, 1, 64, torch.float16)
    q, k = q.abs().contiguous(), k.clone()
    k[3, 0] = float("-inf")
    out = bw.prompt_attention(q, k, v)
    assert torch.isnan(bw.prompt_attention(q[:1], k[3:4], v[3:4])).all()
    keep = torch.arange(70, device="cuda") != 3
    want = torch.cat([bw.prompt_attention(q[i:i + 1], k[:i + 1][keep[:i + 1]], v[:i + 1][keep[:i + 1]]) for i in range(70)])
    assert torch.allclose(out.float(), want.float(), atol=4e-3)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(dtype, scale):
    q, k, v, grad = _inputs(150, 150, 4, 2, 64, dtype, seed=8)
    _check(q, k, v, grad, [(0, 150, 0, 150)], (), 70, 2, scale)


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** 12])
def test_small_and_large_gradients_in_float16_keep_their_bits(size):
    """Products of P and a small gradient lie below float16's steps, those of a large one and the values beyond its range."""
    q, k, v, grad = _inputs(200, 200, 4, 2, 64, torch.float16, seed=9)
    v, grad = (v * (4.0 if size > 1 else 1.0)).contiguous(), grad * size
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = bw.prompt_attention(*leaves)
    got = torch.autograd.grad(out, leaves, grad)
    want = reference(q, k, v, [(0, 200, 0, 200)], None, 0, 64 ** -0.5, grad)
    for name, g, (value, bound) in zip(("dq", "dk", "dv"), got, want[1:]):
        inside = value.abs() < 60000
        # (an upper end of float16 is an infinity; its steps below 2^-14 are 2^-24)
        close(g[inside], value[inside], bound[inside], name)


def test_scores_that_rise_and_fall_over_a_long_axis():
    """The reference is raised again and again: keys grow along the axis, or the largest comes first."""
    for dtype in DTYPES:
        for order in (1, -1):
            q, k, v, grad = _inputs(64, 1500, 2, 1, 64, dtype, seed=3)
            k = (k.float() * torch.linspace(0.1, 4.0, 1500, device="cuda")[::1][:, None, None]).to(dtype)
            k = k if order == 1 else k.flip(0)
            _check(q, k, v, grad, [(0, 64, 0, 1500)], (), None, 0)


def test_gradients_against_differences():
    """Along a direction, from values of the forward itself: inputs are multiples of 2^-6 and the steps 2^-5, exact at both ends.  The outputs' roundings, at most 2^-12 of a value and
    independent, make the difference uncertain by 6 sqrt(2 sum (g y)^2) 2^-12 / 1.7 and the weights' by about as much; the third-order part comes from the 64-bit forward."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, grad = _inputs(90, 120, 4, 2, 64, torch.float16, seed=6)
    q, k, v = ((t.float() * 64).round().div(64).half().contiguous() for t in (q, k, v))
    step = 2.0 ** -5
    d = [torch.randint(0, 2, t.shape, device="cuda", generator=gen) * 2.0 - 1 for t in (q, k, v)]

    def value(s):
        y = bw.prompt_attention(*((t.float() + s * step * u).half() for t, u in zip((q, k, v), d)), window=50, sinks=2)
        return (y.double() * grad.double()).sum(), (y.double() * grad.double()).pow(2).sum()

    def fine(s):
        y = reference(*(t.double() + s * step * u.double() for t, u in zip((q, k, v), d)), [(0, 90, 0, 120)], 50, 2, 0.125)[0][0]
        return (y * grad.double()).sum()

    (up, e1), (down, e2) = value(1), value(-1)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(bw.prompt_attention(*leaves, window=50, sinks=2), leaves, grad)
    along = sum((g.double() * u.double()).sum() for g, u in zip(got, d))
    with torch.no_grad():
        exact = sum((w * u.double()).sum() for (w, _), u in zip(reference(q, k, v, [(0, 90, 0, 120)], 50, 2, 0.125, grad)[1:], d))
    third = (fine(1) - fine(-1)) / (2 * step) - exact
    noise = 2 * 6 * (2 * (e1 + e2)).sqrt() * 2.0 ** -12 / 1.7 / (2 * step)
    own = 6 * sum(((g.double() * u.double()).pow(2).sum()) for g, u in zip(got, d)).sqrt() * 2.0 ** -10
    assert abs((up - down) / (2 * step) - third - along) <= noise + own


def test_streams_captures_and_starts_that_change():
    q, k, v, grad = _inputs(256, 256, 4, 2, 64, torch.bfloat16)
    starts = torch.tensor([0, 100, 256], dtype=torch.int32, device="cuda")
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]

    def step():
        out = bw.prompt_attention(*leaves, starts, window=64, sinks=2)
        return [out, *torch.autograd.grad(out, leaves, grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for cut in (100, 1, 255, 100):
        starts[1] = cut
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), cut
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_autograd_asks():
    q, k, v, grad = _inputs(40, 40, 2, 2, 64, torch.float16)
    full = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(bw.prompt_attention(*full), full, grad)
    for n in range(3):                                           # each gradient alone
        one = [t.detach().clone().requires_grad_(i == n) for i, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(bw.prompt_attention(*one), [one[n]], grad)
        assert torch.equal(g, want[n])
    out = bw.prompt_attention(*full)
    (g,) = torch.autograd.grad(out, [full[0]], grad, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    out = bw.prompt_attention(*full)
    with torch.no_grad():
        full[1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    out = bw.prompt_attention(*full)
    out.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    x = torch.randn(40, 3 * 2 * 64, device="cuda", dtype=torch.float16, requires_grad=True)      # parts of one tensor, one head for all
    a, b, c = x.view(40, 6, 64).split(2, 1)
    bw.prompt_attention(a, b, c).backward(grad)
    assert torch.isfinite(x.grad).all() and x.grad.any()
    with pytest.raises(Exception, match="forward-mode"):
        import torch.autograd.forward_ad as fwd
        with fwd.dual_level():
            bw.prompt_attention(fwd.make_dual(q, torch.ones_like(q)), k, v)


def test_nothing_at_all():
    for shape in ((0, 2, 64), (2, 0, 2, 64), (0, 5, 2, 64)):
        q = torch.zeros(shape, device="cuda", dtype=torch.float16, requires_grad=True)
        kv = torch.zeros(shape, device="cuda", dtype=torch.float16, requires_grad=True)
        out = bw.prompt_attention(q, kv, kv)
        out.sum().backward()
        assert out.shape == q.shape and q.grad.shape == q.shape and kv.grad.shape == kv.shape
    q = torch.randn(5, 2, 64, device="cuda", dtype=torch.float16)
    none = q[:0]
    assert not bw.prompt_attention(q, none, none).any()
    keys = torch.randn(9, 2, 64, device="cuda", dtype=torch.float16, requires_grad=True)
    out = bw.prompt_attention(none, keys, keys)
    out.sum().backward()
    assert not keys.grad.any()


def test_starts_outside_the_tensors_are_their_ends():
    q, k, v, _ = _inputs(50, 50, 2, 1, 64, torch.float16)
    want = bw.prompt_attention(q, k, v, torch.tensor([0, 20, 50], device="cuda"))
    assert torch.equal(bw.prompt_attention(q, k, v, torch.tensor([-7, 20, 2 ** 40], device="cuda")), want)


def test_refusals():
    q, k, v, _ = _inputs(8, 8, 4, 2, 64, torch.float16)
    starts = torch.tensor([0, 8], device="cuda")
    for args, kw, error in (((q, k[:, :, :32], v), {}, ValueError), ((q, k, v[:4]), {}, ValueError), ((q[:, :3], k, v), {}, ValueError), ((q[None], k, v), {}, ValueError),
                            ((q.float(), k, v), {}, TypeError), ((q, k.bfloat16(), v), {}, TypeError), ((q, k, v), {"window": 0}, ValueError), ((q, k, v), {"sinks": -1}, ValueError),
                            ((q, k, v), {"window": 2.5}, TypeError), ((q, k, v, starts[:1]), {}, ValueError), ((q, k, v, starts, starts[None]), {}, ValueError),
                            ((q, k, v, None, starts), {}, ValueError), ((q[None], k[None], v[None], starts), {}, ValueError), ((q, k, v, starts.float()), {}, TypeError),
                            ((q.cpu(), k, v), {}, RuntimeError), ((q, k, v, starts.cpu()), {}, RuntimeError), ((q[..., :60], k[..., :60], v[..., :60]), {}, NotImplementedError)):
        with pytest.raises(error):
            bw.prompt_attention(*args, **kw)
    with pytest.raises(NotImplementedError):
        wide = torch.zeros(2, 1, 264, device="cuda", dtype=torch.float16)
        bw.prompt_attention(wide, wide, wide)
