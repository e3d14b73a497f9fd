"""rotate_heads of arguments that are converted first: leaves stay leaves."""
import pytest
import torch

import bitween_amd as bw

pytestmark = pytest.mark.gpu


def _inputs():
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k = (torch.randn(8, 2, 64, device="cuda", generator=gen).half() for _ in range(2))
    angle = torch.rand(20, 32, device="cuda", generator=gen)
    return q, k, angle.cos(), angle.sin(), torch.randint(0, 20, (8,), device="cuda", generator=gen)


def _weights(layout):
    base = (1 + 0.1 * torch.arange(130, device="cuda") / 130).half()
    w = {"whole": base[:64], "every second": base[:128:2], "off 16 bytes": base[1:65], "parameter": base[:64]}[layout]
    return torch.nn.Parameter(w) if layout == "parameter" else w.detach().requires_grad_(True)


@pytest.mark.parametrize("layout", ["whole", "every second", "off 16 bytes", "parameter"])
@pytest.mark.parametrize("positions", [torch.int64, torch.int32])
def test_weights_of_any_layout_and_their_gradients(positions, layout):
    q, k, cos, sin, pos = _inputs()
    w = _weights(layout)
    plain = w.detach().clone().requires_grad_(True)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    got = bw.rotate_heads(q, k, cos, sin, pos.to(positions), w, w)
    want = bw.rotate_heads(q, k, cos, sin, pos, plain, plain)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.autograd.backward(got, [gq, gk])
    torch.autograd.backward(want, [gq, gk])
    assert torch.equal(w.grad, plain.grad)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out = bw.rotate_heads(q, k, cos, sin, pos.to(positions), w, None)
        with torch.no_grad():
            w.add_(1)
        out[0].sum().backward()


@pytest.mark.parametrize("layout", ["whole", "every second", "off 16 bytes", "parameter"])
@pytest.mark.parametrize("positions", [torch.int64, torch.int32])
def test_a_capture_with_an_eager_graph_of_the_same_leaves_is_refused(positions, layout):
    """Whatever is converted: the accumulation node of a leaf that an eager graph of another stream keeps alive cannot be waited for in a capture."""
    q, k, cos, sin, pos = _inputs()
    pos, leaf = pos.to(positions), _weights(layout)
    alive = bw.rotate_heads(q, k, cos, sin, pos, leaf, None)
    torch.cuda.synchronize()
    graph, refused = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(graph):
        try:
            bw.rotate_heads(q, k, cos, sin, pos, leaf, None)
        except RuntimeError as e:
            refused = str(e)
        out = bw.rotate_heads(q, k, cos, sin, pos, leaf.detach(), None)
    assert refused and "another stream" in refused
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], alive[0])
    torch.autograd.grad(alive[0].float().sum(), leaf)            # the eager graph is as it was
