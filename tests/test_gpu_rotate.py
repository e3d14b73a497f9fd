"""rotate_heads and its gradients against 64 bits, at the sizes and layouts where they can go wrong."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import half_step, rotate

pytestmark = pytest.mark.gpu

SHAPES = [  # tokens, query heads, key heads, dim, rotary
    (1, 32, 32, 128, 128), (7, 12, 12, 64, 64), (33, 8, 2, 80, 80), (5, 3, 1, 80, 40), (129, 32, 8, 128, 64), (61, 5, 5, 96, 96), (17, 4, 4, 256, 256), (3, 1, 1, 8, 8),
    (300, 2, 1, 40, 24), (1031, 8, 8, 128, 128)]


def _inputs(tokens, qh, kh, dim, rotary, dtype, weights, seed=0, table=500):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    angle = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(rotary // 2, device="cuda", dtype=torch.float64) / (rotary // 2))
    fused = torch.randn(tokens, qh + kh + kh, dim, device="cuda", generator=gen).to(dtype)          # rows of a fused projection
    q, k = fused[:, :qh], fused[:, qh:qh + kh]
    w = [(1 + 0.3 * torch.randn(dim, device="cuda", generator=gen)).to(torch.float32 if f32 else dtype) if use else None for use, f32 in weights]
    pos = torch.randint(0, table, (tokens,), device="cuda", generator=gen)
    return q, k, angle.cos().float(), angle.sin().float(), pos, w


def _close(got, want, dtype, slack):
    """One rounding to dtype (below float16's normal range 2^-25), and `slack` for the float32 arithmetic."""
    bound = half_step(dtype) * want.abs() + slack + 2.0 ** -25
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1, f"{worst:.3f} times the bound"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("weights", ["none", "own", "float32", "keys"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, weights, dtype):
    use = {"none": [(0, 0), (0, 0)], "own": [(1, 0), (1, 0)], "float32": [(1, 1), (1, 1)], "keys": [(0, 0), (1, 0)]}[weights]
    q, k, cos, sin, pos, w = _inputs(*shape, dtype, use)
    out = bw.rotate_heads(q, k, cos, sin, pos, w[0], w[1], 1e-5)
    for got, x, weight in zip(out, (q, k), w):
        assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
        want = rotate(x.double(), cos, sin, pos, None if weight is None else weight.double(), 1e-5)
        # a dozen float32 operations on values up to the head's largest, times at most 2 from the sum of two products
        _close(got, want, dtype, 2 * 16 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True).clamp(min=1) * 2)


def test_positions_outside_the_table_are_padding():
    q, k, cos, sin, pos, w = _inputs(40, 4, 2, 64, 64, torch.float16, [(1, 0), (1, 0)], table=50)
    pos[3], pos[17], pos[39] = -1, 50, 2 ** 40
    leaves = [t.clone().requires_grad_(True) for t in (q, k, *w)]
    out = bw.rotate_heads(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[3, 17, 39]] = False
    for o in out:
        assert torch.equal(o[~keep], torch.zeros_like(o[~keep])) and bool((o[keep] != 0).any(-1).all())
    grads = [torch.randn_like(o) for o in out]
    got = torch.autograd.grad(out, leaves, grads)
    short = [t.detach()[keep].clone().requires_grad_(True) for t in leaves[:2]] + [t.detach().clone().requires_grad_(True) for t in leaves[2:]]
    out = bw.rotate_heads(short[0], short[1], cos, sin, pos[keep], short[2], short[3])
    want = torch.autograd.grad(out, short, [g[keep] for g in grads])
    for g, t in zip(got[:2], want[:2]):
        assert torch.equal(g[keep], t) and not g[~keep].any()
    for g, t in zip(got[2:], want[2:]):
        assert torch.allclose(g.float(), t.float(), rtol=2 * half_step(torch.float16), atol=1e-3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("weights", ["none", "own", "float32", "keys"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, weights, dtype):
    use = {"none": [(0, 0), (0, 0)], "own": [(1, 0), (1, 0)], "float32": [(1, 1), (1, 1)], "keys": [(0, 0), (1, 0)]}[weights]
    q, k, cos, sin, pos, w = _inputs(*shape, dtype, use, seed=1)
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (q, k, *w)]
    out = bw.rotate_heads(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3], 1e-5)
    gen = torch.Generator(device="cuda").manual_seed(5)
    grads = [torch.randn(o.shape, device="cuda", generator=gen).to(dtype) for o in out]
    given = [t for t in leaves if t is not None]
    got = dict(zip(map(id, given), torch.autograd.grad(out, given, grads, retain_graph=True)))
    again = torch.autograd.grad(out, given, grads)
    for t, g in zip(given, again):
        assert torch.equal(got[id(t)], g), "the same inputs give the same bits"
    for i in (0, 1):
        x = leaves[i].detach().double().requires_grad_(True)
        weight = None if leaves[2 + i] is None else leaves[2 + i].detach().double().requires_grad_(True)
        y = rotate(x, cos, sin, pos, weight, 1e-5)
        want = torch.autograd.grad(y, [x] if weight is None else [x, weight], grads[i].double())
        # the float32 arithmetic: as above, and the mean of dim products under it; scaled by r (the inputs are near 1, so r is below 3 here)
        scale = want[0].abs().amax(-1, keepdim=True).clamp(min=1) * (1 if weight is None else 3)
        _close(got[id(leaves[i])], want[0], dtype, (2 * 16 + shape[3]) * 2.0 ** -24 * scale * 2)
        if weight is not None:
            n = x.detach() / (x.detach().pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
            back = torch.autograd.grad(rotate(x, cos, sin, pos, None, 1e-5), x, grads[i].double())[0]
            terms = (back * n).abs().sum((0, 1))
            # float32 sums of at most 2^11 terms in a row (a thread's, a block's, the blocks'), each term with 16 roundings
            _close(got[id(leaves[2 + i])], want[1], leaves[2 + i].dtype, (16 + 64) * 2.0 ** -24 * terms)


def test_gradient_against_differences():
    """The derivative along a direction from values of the forward itself.  Inputs are multiples of 2^-6 and the steps 2^-4, so both ends are exact;
    the forward's roundings (at most 2^-12 of a value, independent) make the difference uncertain by 6 times sqrt(2 sum (g y)^2) 2^-12 / 1.7."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, cos, sin, pos, w = _inputs(64, 4, 2, 64, 64, torch.float16, [(1, 0), (1, 0)])
    q, k = ((t.float() * 64).round() / 64 for t in (q, k))
    h = 2.0 ** -4
    dq, dk = (torch.randint(0, 2, t.shape, device="cuda", generator=gen) * 2.0 - 1 for t in (q, k))
    gq, gk = (torch.randn(t.shape, device="cuda", generator=gen).half() for t in (q, k))

    def value(s):
        a, b = bw.rotate_heads((q + s * h * dq).half(), (k + s * h * dk).half(), cos, sin, pos, w[0], w[1])
        return (a.double() * gq.double()).sum() + (b.double() * gk.double()).sum(), (a.double() * gq.double()).pow(2).sum() + (b.double() * gk.double()).pow(2).sum()

    (up, e1), (down, e2) = value(1), value(-1)
    # third-order part of the difference, from the 64-bit forward
    fine = [sum((rotate(x.double() + s * h * d.double(), cos, sin, pos, u.double(), 1e-6) * g.double()).sum() for x, d, g, u in ((q, dq, gq, w[0]), (k, dk, gk, w[1])))
            for s in (1, -1)]
    leaves = [q.half().requires_grad_(True), k.half().requires_grad_(True)]
    a, b = bw.rotate_heads(*leaves, cos, sin, pos, w[0], w[1])
    back = torch.autograd.grad([a, b], leaves, [gq, gk])
    along = (back[0].double() * dq.double()).sum() + (back[1].double() * dk.double()).sum()
    true = [t.double().detach().requires_grad_(True) for t in leaves]
    y = [rotate(x, cos, sin, pos, u.double(), 1e-6) for x, u in zip(true, w)]
    exact = torch.autograd.grad(y, true, [gq.double(), gk.double()])
    curve = (fine[0] - fine[1]) / (2 * h) - ((exact[0] * dq.double()).sum() + (exact[1] * dk.double()).sum())
    noise = 6 * ((e1 + e2).sqrt() * 2.0 ** -12 / 1.7) / (2 * h) + 6 * 2.0 ** -12 * (back[0].double().pow(2).sum() + back[1].double().pow(2).sum()).sqrt()
    assert abs((up - down) / (2 * h) - curve - along) <= noise


def test_layouts():
    """Leading dimensions, transposed heads, expanded tokens, heads of one, and rows that start off 16 bytes give what contiguous rows give."""
    q, k, cos, sin, pos, w = _inputs(24, 4, 4, 64, 64, torch.bfloat16, [(1, 0), (1, 0)])
    q, k = q.contiguous(), k.contiguous()
    want = bw.rotate_heads(q, k, cos, sin, pos, *w)
    got = bw.rotate_heads(q.view(2, 3, 4, 4, 64), k.view(2, 3, 4, 4, 64), cos, sin, pos.view(2, 3, 4), *w)
    assert got[0].shape == (2, 3, 4, 4, 64) and all(torch.equal(a.view(24, 4, 64), b) for a, b in zip(got, want))
    heads_first = [t.view(2, 12, 4, 64).transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]      # strides of [batch, heads, tokens, dim]
    got = bw.rotate_heads(*heads_first, cos, sin, pos.view(2, 12), *w)
    assert all(torch.equal(a.reshape(24, 4, 64), b) for a, b in zip(got, want))
    odd = torch.empty(24, 4, 67, device="cuda", dtype=torch.bfloat16)[..., 1:65]
    odd.copy_(q)
    assert torch.equal(bw.rotate_heads(odd, k, cos, sin, pos, *w)[0], want[0])
    backwards = q.transpose(-1, -2).contiguous().transpose(-1, -2)
    assert torch.equal(bw.rotate_heads(backwards, k, cos, sin, pos, *w)[0], want[0])
    one = k[:, :1].expand(24, 4, 64)
    assert torch.equal(bw.rotate_heads(q, one, cos, sin, pos, *w)[1], bw.rotate_heads(q, one.contiguous(), cos, sin, pos, *w)[1])
    assert all(torch.equal(a, b) for a, b in zip(bw.rotate_heads(q, k, cos.double().half(), sin.half(), pos.int(), *w), bw.rotate_heads(q, k, cos.half().float(), sin.half().float(), pos, *w)))
    none = bw.rotate_heads(q[:0], k[:0], cos, sin, pos[:0], *w)
    assert none[0].shape == (0, 4, 64) and none[1].shape == (0, 4, 64)


def test_gradients_of_shared_expanded_and_unused_outputs():
    q, k, cos, sin, pos, w = _inputs(16, 4, 4, 64, 64, torch.float16, [(1, 0), (1, 0)])
    # the same leaf as queries and keys, and keys broadcast over heads
    x = q.detach().clone().requires_grad_(True)
    a, b = bw.rotate_heads(x, x, cos, sin, pos, *w)
    both, = torch.autograd.grad([a, b], x, [torch.ones_like(a), torch.ones_like(b)])
    ref = x.detach().double().requires_grad_(True)
    want, = torch.autograd.grad(rotate(ref, cos, sin, pos, w[0].double(), 1e-6).sum() + rotate(ref, cos, sin, pos, w[1].double(), 1e-6).sum(), ref)
    assert (both.double() - want).abs().max() <= 3 * half_step(torch.float16) * want.abs().max()        # two roundings and their sum's
    one = k[:, :1].detach().clone().requires_grad_(True)
    y = bw.rotate_heads(q.detach(), one.expand(16, 4, 64), cos, sin, pos, *w)[1]
    got, = torch.autograd.grad(y.sum(), one)                     # (an expanded gradient comes in, the queries' output is unused)
    ref = one.detach().double().requires_grad_(True)
    want, = torch.autograd.grad(rotate(ref.expand(16, 4, 64), cos, sin, pos, w[1].double(), 1e-6).sum(), ref)
    assert got.shape == one.shape and (got.double() - want).abs().max() <= 8 * half_step(torch.float16) * want.abs().max().clamp(min=1)
    # only a weight asks
    u = w[0].detach().clone().requires_grad_(True)
    a, b = bw.rotate_heads(q.detach(), k.detach(), cos, sin, pos, u, w[1])
    assert torch.autograd.grad(a.float().sum() + b.float().sum(), u)[0].shape == (64,)
    # no tokens: a weight's gradient is zero
    a, _ = bw.rotate_heads(q[:0].detach(), k[:0].detach(), cos, sin, pos[:0], u, w[1])
    assert torch.equal(torch.autograd.grad(a.sum(), u)[0], torch.zeros_like(u))


def test_second_derivatives_and_changed_inputs_are_refused():
    q, k, cos, sin, pos, w = _inputs(8, 2, 2, 64, 64, torch.float16, [(1, 0), (1, 0)])
    x = q.detach().clone().requires_grad_(True)
    a, _ = bw.rotate_heads(x, k.detach(), cos, sin, pos, *w)
    g, = torch.autograd.grad(a.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.float().sum().backward()
    a, _ = bw.rotate_heads(x, k.detach(), cos, sin, pos, *w)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        a.float().sum().backward()


def test_captured_forward_and_backward_replayed():
    q, k, cos, sin, pos, w = _inputs(100, 8, 2, 128, 128, torch.bfloat16, [(1, 0), (1, 0)])
    side = torch.cuda.Stream()
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *w)]
    grads = [torch.randn_like(q), torch.randn_like(k)]

    def step():
        out = bw.rotate_heads(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, grads))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            for t in (leaves[0], leaves[1], *grads):
                t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
            pos.copy_(torch.randint(0, 500, pos.shape, device="cuda", generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_a_capture_with_an_eager_graph_of_the_same_leaves_is_refused():
    """The accumulation node of a leaf that an eager graph of another stream keeps alive cannot be waited for in a capture."""
    q, k, cos, sin, pos, w = _inputs(8, 2, 2, 64, 64, torch.float16, [(1, 0), (1, 0)])
    leaf = w[0].detach().clone().requires_grad_(True)
    alive = bw.rotate_heads(q, k, cos, sin, pos, leaf, w[1])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    refused = None
    with torch.cuda.graph(graph):
        try:
            bw.rotate_heads(q, k, cos, sin, pos, leaf, w[1])
        except RuntimeError as e:
            refused = str(e)
        bw.rotate_heads(q, k, cos, sin, pos, leaf.detach(), w[1])
    assert refused and "another stream" in refused
    graph.replay()
    torch.cuda.synchronize()
    torch.autograd.grad(alive[0].float().sum(), leaf)            # the eager graph is as it was


def test_another_stream():
    q, k, cos, sin, pos, w = _inputs(2000, 32, 8, 128, 128, torch.float16, [(1, 0), (1, 0)])
    want = bw.rotate_heads(q, k, cos, sin, pos, *w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bw.rotate_heads(q, k, cos, sin, pos, *w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad
    q, k, cos, sin, pos, _ = _inputs(5, 2, 1, 64, 64, torch.float16, [(0, 0), (0, 0)])
    with fwad.dual_level():
        dual = fwad.make_dual(q, torch.ones_like(q))
        with pytest.raises(RuntimeError):
            bw.rotate_heads(dual, k, cos, sin, pos)
        with torch.no_grad(), pytest.raises(RuntimeError):
            bw.rotate_heads(dual, k, cos, sin, pos)
