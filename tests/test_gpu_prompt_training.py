"""Rotation and attention as a training step runs them together: packed documents, positions of three axes, norms; and captured."""
import pytest
import torch

import bitween_amd as bw

pytestmark = pytest.mark.gpu


def _step(dtype, seed=0, tokens=300, heads=8, kv=2, dim=128):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    fused = torch.randn(tokens, heads + 2 * kv, dim, device="cuda", generator=gen).to(dtype).requires_grad_(True)
    weights = [(1 + 0.2 * torch.randn(dim, device="cuda", generator=gen)).to(dtype).requires_grad_(True) for _ in range(2)]
    angle = torch.arange(400, device="cuda")[:, None] / 10000.0 ** (torch.arange(dim // 2, device="cuda") / (dim // 2))
    positions = torch.randint(0, 400, (3, tokens), device="cuda", generator=gen)
    starts = torch.tensor([0, 17, 170, tokens], device="cuda", dtype=torch.int32)
    grad = torch.randn(tokens, heads, dim, device="cuda", generator=gen).to(dtype)

    def parts():
        return fused.split([heads, kv, kv], 1)

    def rotate(q, k):
        return bw.rotate_heads(q, k, angle.cos(), angle.sin(), positions, *weights, sections=(24, 20, 20), interleaved=True)

    def attend(q, k, v):
        return bw.prompt_attention(q, k, v, starts, window=100, sinks=2)

    return fused, weights, grad, parts, rotate, attend


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_step_is_its_parts(dtype):
    """The gradients through both are those of each, one after the other, bit for bit."""
    fused, weights, grad, parts, rotate, attend = _step(dtype)
    q, k, v = parts()
    out = attend(*rotate(q, k), v)
    whole = torch.autograd.grad(out, [fused, *weights], grad)
    q, k, v = (t.detach().requires_grad_(True) for t in parts())
    turned = [t.detach().requires_grad_(True) for t in rotate(q, k)]
    alone = attend(*turned, v)
    assert torch.equal(alone, out)
    dq, dk, dv = torch.autograd.grad(alone, [*turned, v], grad)
    dx = torch.autograd.grad(rotate(q, k), [q, k, *weights], [dq, dk])
    assert torch.equal(whole[0], torch.cat([dx[0], dx[1], dv], 1)) and torch.equal(whole[1], dx[2]) and torch.equal(whole[2], dx[3])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_captured_step_follows_its_inputs(dtype):
    fused, weights, grad, parts, rotate, attend = _step(dtype)

    def step():
        q, k, v = parts()
        out = attend(*rotate(q, k), v)
        return [out, *torch.autograd.grad(out, [fused, *weights], grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2, 1):
        other = _step(dtype, seed)
        with torch.no_grad():
            for t, o in zip([fused, *weights, grad], [other[0], *other[1], other[2]]):
                t.copy_(o)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        torch.cuda.synchronize()
        del eager


def _layouts(batch, tokens, heads, dim, dtype, gen):
    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)
    return {"heads outside": rand(batch, heads, tokens, dim).transpose(1, 2), "one head for all": rand(batch, tokens, 1, dim).expand(batch, tokens, heads, dim),
            "one sequence for all": rand(1, tokens, heads, dim).expand(batch, tokens, heads, dim), "one token for all": rand(batch, 1, heads, dim).expand(batch, tokens, heads, dim),
            "every second token": rand(batch, 2 * tokens, heads, dim)[:, ::2], "every second value": rand(batch, tokens, heads, 2 * dim)[..., ::2],
            "off 16 bytes": rand(batch * tokens * heads * dim + 1)[1:].view(batch, tokens, heads, dim)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["heads outside", "one head for all", "one sequence for all", "one token for all", "every second token", "every second value", "off 16 bytes"])
def test_layouts_have_the_bits_of_their_copies(layout, dtype):
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v, grad = (_layouts(3, 130, heads, 64, dtype, gen)[layout] for heads in (4, 2, 2, 4))
    got, want = [], []
    for to, change in ((got, lambda t: t), (want, lambda t: t.contiguous().clone())):
        leaves = [change(t).detach().requires_grad_(True) for t in (q, k, v)]
        out = bw.prompt_attention(*leaves, window=50, sinks=1)
        to += [out.detach(), *torch.autograd.grad(out, leaves, change(grad))]
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, want))
