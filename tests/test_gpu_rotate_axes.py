"""rotate_heads with positions of several axes, and its gradients, against 64 bits and against the rotation by one position."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import half_step

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def axis_of(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    n = len(sections)
    return [i % n if i < n * sections[i % n] else 0 for i in range(sum(sections))]


def _table(half, top=300):
    angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] / 1000.0 ** (torch.arange(half, device="cuda", dtype=torch.float64) / half)
    return angle.cos().float(), angle.sin().float()


def _inputs(tokens, heads, kv, dim, sections, dtype, weights, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows = torch.randn(tokens, heads + kv + 1, dim, device="cuda", generator=gen).to(dtype)
    w = [(1 + 0.3 * torch.randn(dim, device="cuda", generator=gen)).to(torch.float32 if f32 else dtype) if use else None for use, f32 in weights]
    positions = torch.randint(0, 300, (len(sections), tokens), device="cuda", generator=gen)
    return rows[:, :heads], rows[:, heads:heads + kv], *_table(sum(sections)), positions, w


def rotate(x, cos, sin, positions, weight, eps, sections, interleaved):
    """x [tokens, heads, dim] float64"""
    half = cos.shape[1]
    y = x if weight is None else x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight
    c, s = (torch.stack([t[positions[a], i] for i, a in enumerate(axis_of(sections, interleaved))], -1).double()[:, None] for t in (cos, sin))
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1)


CASES = [  # tokens, query heads, key heads, dim, sections, interleaved
    (1, 2, 1, 8, (1, 2, 1), False), (7, 4, 4, 64, (16, 8, 8), False), (129, 8, 2, 128, (16, 24, 24), False), (129, 8, 2, 128, (24, 20, 20), True), (33, 5, 1, 80, (13, 27), False),
    (33, 2, 2, 80, (20, 20), True), (17, 4, 1, 128, (5, 0, 27), False), (65, 3, 3, 96, (11, 12, 13, 12), False), (65, 3, 3, 96, (12, 12, 12, 12), True), (40, 2, 1, 256, (128,), False),
    (300, 1, 1, 40, (3, 5, 4), False), (1031, 8, 8, 128, (22, 21, 21), True), (9, 2, 1, 256, (32, 32, 32, 32), True), (9, 2, 1, 64, (30, 1, 1), True)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weights", [[(0, 0), (0, 0)], [(1, 0), (1, 0)], [(0, 0), (1, 1)]])
@pytest.mark.parametrize("case", CASES)
def test_against_64_bits(case, weights, dtype):
    """The bounds of the rotation by one position: one rounding, and 16 float32 operations on values up to the head's largest; for gradients of inputs the mean of dim products too, for
    those of weights sums of at most 2^6 runs of 2^-24 each."""
    tokens, heads, kv, dim, sections, interleaved = case
    q, k, cos, sin, positions, w = _inputs(tokens, heads, kv, dim, sections, dtype, weights)
    kw = dict(eps=1e-5, sections=sections, interleaved=interleaved)
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (q, k, *w)]
    out = bw.rotate_heads(leaves[0], leaves[1], cos, sin, positions, leaves[2], leaves[3], **kw)
    gen = torch.Generator(device="cuda").manual_seed(5)
    grads = [torch.randn(o.shape, device="cuda", generator=gen).to(dtype) for o in out]
    given = [t for t in leaves if t is not None]
    got = torch.autograd.grad(out, given, grads, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(out, given, grads)))
    got = dict(zip(map(id, given), got))
    for i in (0, 1):
        x = leaves[i].detach().double().requires_grad_(True)
        weight = None if w[i] is None else w[i].double().requires_grad_(True)
        y = rotate(x, cos, sin, positions, weight, 1e-5, sections, interleaved)
        assert out[i].is_contiguous() and out[i].dtype == dtype
        slack = 2 * 16 * 2.0 ** -24 * y.detach().abs().amax(-1, keepdim=True).clamp(min=1) * 2
        assert ((out[i].double() - y).abs() <= half_step(dtype) * y.abs() + slack + 2.0 ** -25).all()
        want = torch.autograd.grad(y, [x] if weight is None else [x, weight], grads[i].double())
        scale = want[0].abs().amax(-1, keepdim=True).clamp(min=1)
        if weight is not None:                                   # scaled by the norm's r, which is as large as the smallest head makes it
            scale = scale * 2 * (x.detach().pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt().clamp(min=1)
        assert ((got[id(leaves[i])].double() - want[0]).abs() <= half_step(dtype) * want[0].abs() + (2 * 16 + dim) * 2.0 ** -24 * scale * 2 + 2.0 ** -25).all()
        if weight is not None:
            n = x.detach() / (x.detach().pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
            back = torch.autograd.grad(rotate(x, cos, sin, positions, None, 1e-5, sections, interleaved), x, grads[i].double())[0]
            g = got[id(leaves[2 + i])]
            assert ((g.double() - want[1]).abs() <= half_step(g.dtype) * want[1].abs() + (16 + 64) * 2.0 ** -24 * (back * n).abs().sum((0, 1)) + 2.0 ** -25).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_equal_positions_are_one_position(interleaved):
    q, k, cos, sin, positions, w = _inputs(100, 4, 2, 128, (24, 20, 20), torch.bfloat16, [(1, 0), (1, 0)])
    one = positions[0]
    want = bw.rotate_heads(q, k, cos, sin, one, *w)
    got = bw.rotate_heads(q, k, cos, sin, one.expand(3, -1), *w, sections=[24, 20, 20], interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    single = bw.rotate_heads(q, k, cos, sin, one[None], *w, sections=(64,))
    assert all(torch.equal(a, b) for a, b in zip(single, want))


def test_a_position_outside_on_any_axis_is_padding():
    q, k, cos, sin, positions, w = _inputs(30, 4, 2, 64, (16, 8, 8), torch.float16, [(1, 0), (1, 0)])
    positions[0, 3], positions[1, 7], positions[2, 29] = -1, 300, 2 ** 40
    leaves = [t.clone().requires_grad_(True) for t in (q, k, *w)]
    out = bw.rotate_heads(leaves[0], leaves[1], cos, sin, positions, leaves[2], leaves[3], sections=(16, 8, 8))
    pad = torch.zeros(30, dtype=torch.bool, device="cuda")
    pad[[3, 7, 29]] = True
    grads = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    for t in (*out, *grads[:2]):
        assert not t[pad].any() and t[~pad].any(-1).all()
    # nothing of them in the weights' gradients either
    keep = [t.detach()[~pad].clone().requires_grad_(True) for t in leaves[:2]] + [t.detach().clone().requires_grad_(True) for t in leaves[2:]]
    short = bw.rotate_heads(keep[0], keep[1], cos, sin, positions[:, ~pad], keep[2], keep[3], sections=(16, 8, 8))
    for a, b in zip(grads[2:], torch.autograd.grad(short, keep[2:], [torch.ones_like(o) for o in short])):
        assert torch.allclose(a.float(), b.float(), rtol=2 * half_step(torch.float16), atol=1e-3)


def test_leading_dimensions_streams_and_captures():
    q, k, cos, sin, positions, w = _inputs(60, 4, 2, 64, (16, 8, 8), torch.float16, [(1, 0), (1, 0)])
    want = bw.rotate_heads(q, k, cos, sin, positions, *w, sections=(16, 8, 8))
    got = bw.rotate_heads(q.unflatten(0, (3, 20)), k.unflatten(0, (3, 20)), cos, sin, positions.view(3, 3, 20), *w, sections=(16, 8, 8))
    assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, want))
    got = bw.rotate_heads(q, k, cos, sin, positions.to(torch.int32), *w, sections=(16, 8, 8))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bw.rotate_heads(q, k, cos, sin, positions, *w, sections=(16, 8, 8))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = bw.rotate_heads(q, k, cos, sin, positions, *w, sections=(16, 8, 8))
    for _ in range(3):
        positions.copy_((positions * 7 + 1) % 300)
        graph.replay()
        torch.cuda.synchronize()
        eager = bw.rotate_heads(q, k, cos, sin, positions, *w, sections=(16, 8, 8))
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        torch.cuda.synchronize()


def test_refusals():
    q, k, cos, sin, positions, _ = _inputs(6, 2, 1, 64, (16, 8, 8), torch.float16, [(0, 0), (0, 0)])
    for at, kw, error in ((positions, dict(sections=(16, 8)), ValueError), (positions, dict(sections=(16, 8, 7)), ValueError), (positions, dict(sections=(40, -8, 0)), ValueError),
                          (positions, dict(sections=(8, 8, 8, 4, 4)), ValueError), (positions, dict(sections=(8, 16, 8), interleaved=True), ValueError),
                          (positions[0], dict(interleaved=True), ValueError), (positions, dict(sections=(16.0, 8, 8)), TypeError), (positions, dict(sections=16), TypeError),
                          (positions, dict(sections=(16, 8, 8), interleaved=1), TypeError), (positions[:2], dict(sections=(16, 8, 8)), ValueError), (positions, {}, ValueError),
                          (positions[:, :5], dict(sections=(16, 8, 8)), ValueError), (positions.float(), dict(sections=(16, 8, 8)), TypeError)):
        with pytest.raises(error):
            bw.rotate_heads(q, k, cos, sin, at, **kw)
