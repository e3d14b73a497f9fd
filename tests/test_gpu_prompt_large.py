"""Prompts, appends and windows whose offsets pass 32 bits, two captured graphs of them, and a capture that is refused."""
import pytest
import torch

import bitween_amd as bw

pytestmark = pytest.mark.gpu


def _room(size):
    if torch.cuda.mem_get_info()[0] < size:
        pytest.skip(f"{size / 1e9:.0f} GB of memory")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_that_lie_gigabytes_apart(dtype):
    """Rows of one tensor, nearly 2^24 elements each (32 MB), 200 of them: the same bits as their copies."""
    _room(12e9)
    big = torch.empty(200, 2 ** 24 - 64, device="cuda", dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(0)
    big[:, -1024:] = torch.randn(200, 1024, device="cuda", generator=gen).to(dtype)
    k, v, q, grad = (big[:, -1024 + a:-1024 + b].unflatten(1, (-1, 64)) for a, b in ((0, 64), (64, 128), (128, 384), (384, 640)))
    got, want = [], []
    for to, change in ((got, lambda t: t), (want, lambda t: t.contiguous())):
        leaves = [change(t).detach().requires_grad_(True) for t in (q, k, v)]
        out = bw.prompt_attention(*leaves, window=90, sinks=3)
        to += [out.detach(), *torch.autograd.grad(out, leaves, change(grad))]
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, want))
    del big, k, v, q, grad, leaves, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64)])
def test_pages_behind_four_gigabytes(bits, group):
    """The last pages of a cache of 4.5 GB of keys, against a cache of those pages alone."""
    _room(14e9)
    kv, dim, page, length = 8, 128, 64, 500
    per_page = page * kv * dim * bits // 8
    pages, used = 4_500_000_000 // per_page, -(-length // page)
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(length, 16, dim, device="cuda", generator=gen).half()
    k, v = (torch.randn(length, kv, dim, device="cuda", generator=gen).half() for _ in range(2))
    angle = torch.arange(length, device="cuda")[:, None] / 10000.0 ** (torch.arange(dim // 2, device="cuda") / (dim // 2))
    cos, sin, at = angle.cos(), angle.sin(), torch.arange(length, device="cuda")
    results = []
    for count in (pages, used):
        cache = bw.PagedCache(count, kv, dim, page, bits, group)
        table = torch.arange(count - used, count, device="cuda", dtype=torch.int32)[None]
        slots = cache.slots(table, at, torch.zeros_like(at))
        turned = cache.append(q, k, v, cos, sin, at, slots)
        lengths = torch.tensor([length], device="cuda", dtype=torch.int32)
        results.append([turned, *cache.read(slots), cache.attend(turned[-1:], table, lengths, window=200, sinks=5)])
        del cache
        torch.cuda.empty_cache()
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_two_graphs_and_eager_calls_in_turn():
    """Each has workspaces of its own: parts of a long axis, pieces of the keys' gradients."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    sets = []
    for tokens, dtype in ((30, torch.float16), (1200, torch.bfloat16)):
        q = torch.randn(tokens, 8, 64, device="cuda", generator=gen).to(dtype)
        k, v = (torch.randn(6000 if tokens == 30 else tokens, 2, 64, device="cuda", generator=gen).to(dtype) for _ in range(2))
        sets.append(([t.requires_grad_(True) for t in (q, k, v)], torch.randn_like(q)))

    def step(leaves, grad):
        out = bw.prompt_attention(*leaves)
        return [out, *torch.autograd.grad(out, leaves, grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[t.detach().clone() for t in step(*s)] for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(step(*s))
    for _ in range(3):
        for g in graphs:
            g.replay()
        eager = [[t.detach().clone() for t in step(*s)] for s in sets]
        torch.cuda.synchronize()
        for w, a, b in zip(want, got, eager):
            assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(w, a, b))
        for a in got:
            for t in a:
                t.detach().zero_()


def test_a_capture_with_an_eager_graph_of_the_same_leaves_is_refused():
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(40, 2, 64, device="cuda", generator=gen).half() for _ in range(3))
    for n in range(3):
        leaves = [t.detach().requires_grad_(i == n) for i, t in enumerate((q, k, v))]
        alive = bw.prompt_attention(*leaves)
        torch.cuda.synchronize()
        graph, refused = torch.cuda.CUDAGraph(), None
        with torch.cuda.graph(graph):
            try:
                bw.prompt_attention(*leaves)
            except RuntimeError as e:
                refused = str(e)
            out = bw.prompt_attention(q, k, v)
        assert refused and "another stream" in refused
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, alive.detach())
