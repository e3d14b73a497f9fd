"""rotate_heads beyond the 2^32 threads of one launch."""
import pytest
import torch

import bitween_amd as bw

pytestmark = pytest.mark.gpu


def test_more_threads_than_a_launch_has():
    """Heads of 136 values have 17 lanes, filled up to 32: 2^26 + 5 tokens of two heads are 2^32 + 320 threads.  The inputs are 64 tokens over and over
    (an expanded view), so that every token's result is that of its residue; 37 GB of results."""
    tokens, period, dim = 2 ** 26 + 5, 64, 136
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("60 GB of memory")
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, 2, dim, device="cuda", generator=gen).half()
    angle = torch.rand(period, dim // 2, device="cuda", generator=gen)
    cos, sin = angle.cos(), angle.sin()
    positions = torch.arange(tokens, device="cuda") % period
    want = bw.rotate_heads(x[:, :1].expand(period, 1, dim), x[:, 1:].expand(period, 1, dim), cos, sin, positions[:period])
    got = bw.rotate_heads(x[:, :1].expand(tokens, 1, dim), x[:, 1:].expand(tokens, 1, dim), cos, sin, positions)
    for g, w in zip(got, want):
        whole = tokens // period * period
        for at in range(0, whole, 2 ** 22):
            part = g[at:min(at + 2 ** 22, whole)].view(-1, period, 1, dim)
            assert bool((part == w).all()), f"tokens from {at} on"
        assert torch.equal(g[whole:], w[:tokens - whole])
    del got, g, part
    torch.cuda.empty_cache()
