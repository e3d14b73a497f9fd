"""append_cache against rotate_heads and write_cache, and against 64 bits where a norm's last bit is its own."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import half_step, quantize, unpack
from test_gpu_rotate_axes import rotate

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _inputs(tokens, heads, kv, dim, rotary, dtype, weights=False, axes=None, seed=0, top=400):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    half = rotary // 2
    angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] / 1000.0 ** (torch.arange(half, device="cuda", dtype=torch.float64) / half)
    rows = torch.randn(tokens, heads + 2 * kv, dim, device="cuda", generator=gen).to(dtype)
    w = [(1 + 0.3 * torch.randn(dim, device="cuda", generator=gen)).to(dtype) if weights else None for _ in range(2)]
    positions = torch.randint(0, top, (len(axes), tokens) if axes else (tokens,), device="cuda", generator=gen)
    return [rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:], angle.cos().float(), angle.sin().float(), positions], w


def _cache(kv, dim, bits, group, page, dtype, tokens, seed=0):
    pages = -(-tokens // page) + 2
    cache = bw.PagedCache(pages, kv, dim, page, bits, group, dtype)
    for t in (cache.keys, cache.values, cache.key_meta, cache.value_meta):
        if t is not None:
            t.view(torch.uint8).random_(0, 100, generator=torch.Generator(device="cuda").manual_seed(seed))
    return cache, torch.randperm(pages * page, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 1))[:tokens]


def _tensors(cache):
    return [t for t in (cache.keys, cache.values, cache.key_meta, cache.value_meta) if t is not None]


CASES = [  # tokens, query heads, key heads, dim, rotary, group, page, sections
    (1, 32, 32, 128, 128, 64, 16, None), (5, 4, 2, 64, 64, 32, 16, None), (33, 8, 2, 96, 96, 32, 32, None), (70, 3, 1, 128, 64, 128, 64, None), (129, 5, 5, 64, 32, 64, 16, (4, 6, 6)),
    (64, 16, 1, 256, 256, 128, 16, None), (40, 2, 2, 160, 160, 32, 128, (20, 30, 30)), (300, 8, 8, 128, 128, 32, 16, (16, 24, 24)), (31, 2, 1, 64, 40, 32, 16, None), (12, 1, 1, 192, 128, 64, 16, None),
    (9, 2, 3, 32, 32, 32, 16, None)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("case", CASES)
def test_without_norms_it_is_the_two_calls(case, bits, dtype):
    tokens, heads, kv, dim, rotary, group, page, sections = case
    if heads % kv:
        heads = kv * heads
    (q, k, v, cos, sin, positions), _ = _inputs(tokens, heads, kv, dim, rotary, dtype, axes=sections)
    # padding: by its slot, by its position, by both
    cache, slots = _cache(kv, dim, bits, group, page, dtype, tokens)
    if tokens > 8:
        slots[2], slots[5] = -1, 2 ** 40
        positions[..., 3], positions[..., 5] = -1, 400
    plain = bw.PagedCache(cache.keys.shape[0], kv, dim, page, bits, group, dtype)
    for a, b in zip(_tensors(plain), _tensors(cache)):
        a.copy_(b)
    got = cache.append(q, k, v, cos, sin, positions, slots, sections=sections)
    want, rotated = bw.rotate_heads(q, k, cos, sin, positions, sections=sections)
    inside = ((positions >= 0) & (positions < 400)).view(-1, tokens).all(0)
    plain.write(rotated, v, torch.where(inside, slots, -1))
    assert torch.equal(got, want) and got.is_contiguous()
    for a, b in zip(_tensors(cache), _tensors(plain)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64), (8, 128), (4, 32)])
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,sections", [(3, 8, 2, 128, 128, None), (200, 4, 4, 128, 64, None), (65, 2, 1, 256, 256, (40, 44, 44))])
def test_norms(tokens, heads, kv, dim, rotary, sections, bits, group, dtype):
    """The root is the nearest float32 (but for one of 2^28 values next to half a step), the rest single float32 operations that are done here in the same order: the same bits as
    float32 tensors give on the host."""
    (q, k, v, cos, sin, positions), w = _inputs(tokens, heads, kv, dim, rotary, dtype, weights=True, axes=sections, seed=3)
    cache, slots = _cache(kv, dim, bits, group or 64, 16, dtype, tokens)
    got = cache.append(q, k, v, cos, sin, positions, slots, *w, 1e-5, sections=sections)
    at = [a for a, n in enumerate(sections) for _ in range(n)] if sections else None
    half = rotary // 2
    c, s = ((t[positions] if at is None else torch.stack([t[positions[a], i] for i, a in enumerate(at)], -1)).cpu()[:, None] for t in (cos, sin))

    def turned(x, weight):
        x = x.cpu()
        eps = torch.tensor(1e-5).double()                        # (a float32)
        r = (x.double().pow(2).mean(-1, keepdim=True) + eps).pow(-0.5).float()
        y = x.float() * r * weight.cpu().float()
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1).to(x.dtype)

    assert torch.equal(got.cpu(), turned(q, w[0]))
    exact = rotate(q.double(), cos, sin, positions if sections else positions[None], w[0].double(), 1e-5, sections or (half,), False)
    assert ((got.double() - exact).abs() <= half_step(dtype) * exact.abs() + 64 * 2.0 ** -24 * exact.abs().amax(-1, keepdim=True).clamp(min=1) + 2.0 ** -25).all()
    page, row = slots // 16, slots % 16
    for x, words, meta in ((turned(k, w[1]), cache.keys, cache.key_meta), (v.cpu(), cache.values, cache.value_meta)):
        if bits == 16:
            assert torch.equal(words[page, :, row].cpu(), x)
            continue
        codes, scale, zero = quantize(x.double().numpy(), bits, group)
        assert (unpack(words[page, :, row].cpu().numpy(), bits, dim) == codes).all()
        pairs = meta[page, :, :, row].cpu().numpy()
        assert (pairs[..., 0] == scale).all() and (pairs[..., 1] == zero).all()


def test_infinities_and_nan_mark_their_group():
    (q, k, v, cos, sin, positions), _ = _inputs(20, 2, 2, 128, 64, torch.float16)
    k, v = k.clone(), v.clone()
    k[3, 1, 5], v[4, 0, 100] = float("inf"), float("nan")
    cache, slots = _cache(2, 128, 8, 32, 16, torch.float16, 20)
    cache.append(q, k, v, cos, sin, positions, slots)
    for got, bad in zip(cache.read(slots), ({(3, 1, 0), (3, 1, 1)}, {(4, 0, 3)})):      # the pair turns: both halves of the rotation
        nan = torch.isnan(got).unflatten(-1, (4, 32)).any(-1).nonzero().tolist()
        assert set(map(tuple, nan)) == bad


def test_rows_of_the_cache_itself():
    cache = bw.PagedCache(2, 2, 64, 16, 16, dtype=torch.float16)
    cache.keys.normal_()
    cache.values.normal_()
    (_, _, _, cos, sin, positions), _ = _inputs(16, 2, 2, 64, 64, torch.float16)
    k, v = cache.keys[0].transpose(0, 1), cache.values[0].transpose(0, 1)
    want = bw.rotate_heads(k.clone(), k.clone(), cos, sin, positions)
    old = v.clone()
    slots = torch.arange(16, device="cuda").flip(0)
    got = cache.append(k, k, v, cos, sin, positions, slots)
    assert torch.equal(got, want[0])
    assert torch.equal(cache.keys[0].transpose(0, 1)[slots], want[1]) and torch.equal(cache.values[0].transpose(0, 1)[slots], old)


def test_other_layouts_streams_and_captures():
    (q, k, v, cos, sin, positions), w = _inputs(48, 4, 2, 64, 64, torch.bfloat16, weights=True)
    cache, slots = _cache(2, 64, 8, 32, 16, torch.bfloat16, 48)
    before = [t.clone() for t in _tensors(cache)]
    want = cache.append(q, k, v, cos, sin, positions, slots, *w)
    after = [t.clone() for t in _tensors(cache)]

    def again(f):
        for t, b in zip(_tensors(cache), before):
            t.copy_(b)
        got = f()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and all(torch.equal(t, a) for t, a in zip(_tensors(cache), after))

    again(lambda: cache.append(q.contiguous(), k.transpose(0, 1).contiguous().transpose(0, 1), torch.nn.functional.pad(v, (0, 3))[..., :64], cos, sin, positions.int(), slots.int(), *w))
    again(lambda: cache.append(q, k, v, cos, sin, positions, slots, w[0][None].expand(2, -1)[1], torch.cat([w[1].new_zeros(1), w[1]])[1:]))
    side = torch.cuda.Stream()

    def on_side():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = cache.append(q, k, v, cos, sin, positions, slots, *w)
        torch.cuda.current_stream().wait_stream(side)
        return got

    again(on_side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = cache.append(q, k, v, cos, sin, positions, slots, *w)
    for _ in range(3):
        again(lambda: (graph.replay(), captured)[1])
    version = cache.keys._version
    cache.append(q, k, v, cos, sin, positions, slots, *w)
    assert cache.keys._version == version + 1


def test_nothing_to_append():
    cache = bw.PagedCache(2, 2, 64, 16, 16)
    (q, k, v, cos, sin, positions), _ = _inputs(4, 4, 2, 64, 64, torch.float16)
    out = cache.append(q[:0], k[:0], v[:0], cos, sin, positions[:0], positions[:0])
    assert out.shape == (0, 4, 64) and not cache.keys.any()


def test_refusals():
    cache = bw.PagedCache(2, 2, 64, 16, 16)
    (q, k, v, cos, sin, positions), w = _inputs(4, 4, 2, 64, 64, torch.float16, weights=True)
    slots = torch.arange(4, device="cuda")
    good = [q, k, v, cos, sin, positions, slots]
    cache.append(*good)
    for i, bad, error in ((0, q.bfloat16(), TypeError), (0, q[0], ValueError), (0, q[..., :32], ValueError), (1, k[:, :1], ValueError), (2, v[:3], ValueError), (2, v.bfloat16(), TypeError),
                          (3, cos[:, :3], ValueError), (5, positions[:3], ValueError), (5, positions.float(), TypeError), (6, slots[:3], ValueError), (6, slots.float(), TypeError),
                          (0, q.cpu(), RuntimeError), (6, slots.cpu(), RuntimeError), (0, q.clone().requires_grad_(True), bw.kernels.hip_loader.BitweenHipError),
                          (2, v.clone().requires_grad_(True), bw.kernels.hip_loader.BitweenHipError)):
        with pytest.raises(error):
            cache.append(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError):
        cache.append(*good, sections=(16, 16))
    with pytest.raises(ValueError):
        cache.append(*good, w[0][:32], None)
    with pytest.raises(TypeError):
        bw.append_cache(*(t.bfloat16() if n < 3 else t for n, t in enumerate(good)), cache.keys, cache.values)
    shared = torch.zeros(2, 2, 16, 64, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        bw.append_cache(*good, shared, shared)
    with torch.no_grad():
        cache.append(q.clone().requires_grad_(True), *good[1:])
