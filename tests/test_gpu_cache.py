"""The paged key-value cache: what is written and read back, bit for bit against the format's definition."""
import numpy as np
import pytest
import torch

import bitween_amd as bw
from attention_ref import quantize, rows, unpack

pytestmark = pytest.mark.gpu

FORMATS = [(16, 0), (8, 32), (8, 64), (8, 128), (4, 32), (4, 64), (4, 128)]


def _cache(pages, heads, dim, page, bits, group, dtype):
    c = bw.PagedCache(pages, heads, dim, page, bits, group or 64, dtype)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for t in (c.keys, c.values, c.key_meta, c.value_meta):
        if t is not None:
            t.view(torch.int16).random_(-2 ** 15, 2 ** 15 - 1, generator=gen) if t.dtype != torch.int32 else t.random_(-2 ** 31, 2 ** 31 - 1, generator=gen)
    return c


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def _check(c, x, slots, words, meta):
    """Codes, scales and zero points of the rows, and the values read back."""
    page, row = slots // c.page_size, slots % c.page_size
    if c.bits == 16:
        assert torch.equal(_bits(words[page, :, row]), _bits(x))
        return
    codes, scale, zero = quantize(x.double().cpu().numpy(), c.bits, c.group_size)
    bad = np.isnan(scale)
    pairs = meta[page, :, :, row].cpu().numpy()
    assert np.array_equal(np.isnan(pairs[..., 0]), bad) and np.array_equal(pairs[..., 0][~bad], scale[~bad])
    assert np.array_equal(pairs[..., 1][~bad].astype(np.float64), zero[~bad])
    got = unpack(words[page, :, row].cpu().numpy(), c.bits, x.shape[-1])
    keep = np.repeat(~bad, c.group_size, -1)
    assert np.array_equal(got[keep], codes[keep])


def _check_read(c, slots, out, words, meta):
    want = rows(words, meta, slots, c.bits, c.group_size)
    if out.dtype == torch.float16 and c.bits != 16:
        want = want.clamp(-65504, 65504)
    want = want.to(out.dtype)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(_bits(torch.nan_to_num(out)), _bits(torch.nan_to_num(want)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 32, 128, 16), (37, 3, 128, 64), (130, 1, 256, 1024), (1000, 8, 128, 32), (5, 2, 384 // 2, 128)])
def test_write_and_read(tokens, heads, dim, page, bits, group, dtype):
    if group and dim % group:
        pytest.skip("the group does not divide this head")
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    pages = -(-tokens // page) + 3
    c = _cache(pages, heads, dim, page, bits, group, dtype)
    before = [None if t is None else t.clone() for t in (c.keys, c.values, c.key_meta, c.value_meta)]
    fused = torch.randn(tokens, 2 * heads, dim, device="cuda", generator=gen)
    fused *= 10.0 ** torch.randint(-3, 3, (tokens, 2 * heads, 1), device="cuda", generator=gen)
    fused = (fused + torch.randint(-2, 3, (tokens, 2 * heads, 1), device="cuda", generator=gen)).to(dtype)      # one-sided groups among them
    k, v = fused[:, :heads], fused[:, heads:]
    slots = torch.randperm(pages * page, device="cuda", generator=gen)[:tokens]
    c.write(k, v, slots)
    for x, words, meta in ((k, c.keys, c.key_meta), (v, c.values, c.value_meta)):
        _check(c, x, slots, words, meta)
    # no other row has changed
    others = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    others[slots] = False
    others = others.nonzero()[:, 0]
    for now, old in zip((c.keys, c.values, c.key_meta, c.value_meta), before):
        if now is not None:
            n, o = (t.transpose(2, 3) if t.dim() == 5 else t for t in (now, old))          # pairs: [pages, heads, page, groups, 2]
            at = (others // page, slice(None), others % page)
            assert torch.equal(_bits(n[at]), _bits(o[at]))
    out = c.read(slots)
    for got, x, words, meta in zip(out, (k, v), (c.keys, c.values), (c.key_meta, c.value_meta)):
        assert got.shape == x.shape and got.dtype == dtype
        _check_read(c, slots, got, words, meta)
        if bits != 16:                                           # within half a scale of what was written
            pairs = meta[slots // page, :, :, slots % page].double()
            exact = rows(words, meta, slots, bits, c.group_size)
            assert bool(((exact - x.double()).abs().unflatten(-1, (-1, c.group_size)) <= pairs[..., :1] / 2).all())


def _special(dtype, dim):
    """Rows whose groups are hard: zeros, one value, one-sided, ties, tiny, the largest finite values, infinities and NaN."""
    big = torch.finfo(dtype).max
    t = torch.arange(dim, dtype=torch.float64)
    halves = (t % 31) - 15 + 0.5
    return torch.stack([torch.zeros(dim), torch.full((dim,), 3.0), torch.full((dim,), -0.3), 5 + t / dim, -5 - t / dim, halves, torch.where(t == 0, 15.0, halves),
                        torch.where(t == 0, 255.0, torch.where(t == 1, 0.0, halves.abs())), t * 2.0 ** -24, torch.where(t % 2 == 0, 2.0 ** -24, 0.0),
                        torch.where(t == 3, big, 0.0), torch.where(t % 2 == 0, big, -big), torch.where(t == 1, float("inf"), 1.0),
                        torch.where(t == dim - 1, float("nan"), -1.0), torch.where(t == 0, -float("inf"), t), -0.0 * t, t * 1e-4 - 3e-3]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits,group", FORMATS)
def test_hard_groups(bits, group, dtype):
    x = _special(dtype, 128).cuda()[:, None].expand(-1, 2, -1)
    c = _cache(3, 2, 128, 16, bits, group, dtype)
    slots = torch.arange(x.shape[0], device="cuda") * 2 + 1
    c.write(x, x.flip(0), slots)
    _check(c, x, slots, c.keys, c.key_meta)
    _check(c, x.flip(0), slots, c.values, c.value_meta)
    for got, words, meta in zip(c.read(slots), (c.keys, c.values), (c.key_meta, c.value_meta)):
        _check_read(c, slots, got, words, meta)
        assert bits == 16 or not torch.isinf(got).any()


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64), (4, 32)])
def test_slots_outside_the_cache_are_padding(bits, group):
    c = _cache(4, 2, 64, 16, bits, group, torch.float16)
    before = [None if t is None else t.clone() for t in (c.keys, c.values, c.key_meta, c.value_meta)]
    x = torch.randn(5, 2, 64, device="cuda").half()
    c.write(x, x, torch.tensor([-1, 64, 2 ** 40, -2 ** 62, 10 ** 6], device="cuda"))
    for now, old in zip((c.keys, c.values, c.key_meta, c.value_meta), before):
        assert now is None or torch.equal(_bits(now), _bits(old))
    slots = torch.tensor([-1, 3, 64, 5, -7], device="cuda")
    c.write(x, -x, slots)
    k, v = c.read(slots)
    for got, words, meta in ((k, c.keys, c.key_meta), (v, c.values, c.value_meta)):
        assert not got[[0, 2, 4]].any()
        _check_read(c, slots[[1, 3]], got[[1, 3]], words, meta)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    c.write(x[:0], x[:0], none)
    assert c.read(none)[0].shape == (0, 2, 64)


def test_small_and_odd_heads_at_16_bits_and_layouts():
    for dim in (8, 40, 80, 120):
        c = _cache(2, 3, dim, 16, 16, 0, torch.bfloat16)
        x = torch.randn(7, 3, dim, device="cuda").bfloat16()
        slots = torch.tensor([31, 0, 16, 15, 2, 9, 30], device="cuda")
        c.write(x, -x, slots)
        assert torch.equal(c.read(slots)[0], x) and torch.equal(c.read(slots)[1], -x)
    c = _cache(4, 4, 64, 16, 8, 64, torch.float16)
    base = torch.randn(20, 4, 64, device="cuda").half()
    slots = torch.randperm(64, device="cuda")[:20]
    c.write(base, base, slots)
    want = c.keys.clone(), c.key_meta.clone()
    heads_first = base.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(20, 4, 67, device="cuda", dtype=torch.float16)[..., 1:65].copy_(base)
    across = base.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (heads_first, odd, across):
        c.keys.zero_(), c.key_meta.zero_()
        c.write(x, base, slots.int())                            # (slots of another whole-number type are converted)
        got = c.read(slots)[0]
        page, row = slots // 16, slots % 16
        assert torch.equal(c.keys[page, :, row], want[0][page, :, row]) and torch.equal(c.key_meta[page, :, :, row], want[1][page, :, :, row])
        assert torch.equal(got, bw.read_cache(slots, want[0], c.values, want[1], c.value_meta, 8, 64)[0])
    assert bw.read_cache(slots, c.keys, c.values, c.key_meta, c.value_meta, 8, 64, torch.bfloat16)[0].dtype == torch.bfloat16


def test_a_write_is_seen_by_autograd_and_by_other_streams():
    c = _cache(4, 2, 64, 16, 16, 0, torch.float16)
    version = c.keys._version, c.values._version
    x = torch.randn(3, 2, 64, device="cuda").half()
    slots = torch.tensor([5, 1, 40], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.write(x, x, slots)
        got = c.read(slots)
    torch.cuda.current_stream().wait_stream(side)
    assert c.keys._version > version[0] and c.values._version > version[1]
    assert torch.equal(got[0], x)


@pytest.mark.parametrize("bits,group", [(16, 0), (4, 64)])
def test_captured_and_replayed(bits, group):
    c = _cache(8, 2, 64, 16, bits, group, torch.float16)
    x, slots = torch.randn(6, 2, 64, device="cuda").half(), torch.arange(6, device="cuda")
    c.write(x, x, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.write(x, -x, slots)
        out = c.read(slots)
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        slots.copy_(torch.randperm(128, device="cuda", generator=gen)[:6])
        graph.replay()
        torch.cuda.synchronize()
        _check(c, x, slots, c.keys, c.key_meta)
        for a, b in zip(out, c.read(slots)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 128)])
def test_rows_behind_four_gibibytes(bits, group):
    """Offsets of rows and pairs beyond 32 bits, in bytes and in elements: 2.4 billion values of keys."""
    pages = 2304
    c = bw.PagedCache(pages, 8, 128, 1024, bits, group or 64, torch.float16)
    x = torch.randn(40, 8, 128, device="cuda").half()
    slots = torch.cat([torch.arange(20, device="cuda"), pages * 1024 - 1 - torch.arange(20, device="cuda") * 50000])
    c.write(x, -x, slots)
    _check(c, x, slots, c.keys, c.key_meta)
    _check(c, -x, slots, c.values, c.value_meta)
    k, v = c.read(slots)
    _check_read(c, slots, k, c.keys, c.key_meta)
    # the last page of the cache as a sequence of its own
    table = torch.tensor([[pages - 1], [0]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 16, 128, device="cuda").half()
    out = c.attend(q, table, torch.tensor([1024, 20], dtype=torch.int32, device="cuda"))
    for b, (page, n) in enumerate(((pages - 1, 1024), (0, 20))):
        at = page * 1024 + torch.arange(n, device="cuda")
        kk, vv = (rows(w, m, at, bits, c.group_size).transpose(0, 1).contiguous() for w, m in ((c.keys, c.key_meta), (c.values, c.value_meta)))
        scores = torch.matmul(q[b].double().view(8, 2, 128), kk.transpose(1, 2).contiguous()) * 128 ** -0.5
        want = torch.matmul(torch.softmax(scores, -1), vv).reshape(16, 128)
        assert (out[b].double() - want).abs().max() <= 2.0 ** -11 * want.abs().max() + 2.0 ** -15 * vv.abs().max()
    if bits != 16:
        at = torch.arange(20, device="cuda")
        _check_read(c, at, bw.read_cache(at, c.keys, c.values, c.key_meta, c.value_meta, bits, group)[0], c.keys, c.key_meta)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_of_the_cache_itself_may_be_written(dtype):
    """Every row of a page one row further on, and pages the other way round: what is read is what was there before the call."""
    c = _cache(4, 2, 64, 1024, 16, 0, dtype)
    c.keys.copy_(torch.randn(c.keys.shape, device="cuda"))
    c.values.copy_(torch.randn(c.values.shape, device="cuda"))
    k, v = c.keys.clone(), c.values.clone()
    c.write(c.keys[1].transpose(0, 1)[:1023], c.values[1].transpose(0, 1)[:1023], torch.arange(1025, 2048, device="cuda"))
    for got, was in ((c.keys, k), (c.values, v)):
        assert torch.equal(got[1, :, 1:], was[1, :, :1023]) and torch.equal(got[1, :, 0], was[1, :, 0])
        assert torch.equal(got[[0, 2, 3]], was[[0, 2, 3]])


def test_keys_and_values_in_one_place_are_refused():
    c = _cache(2, 2, 64, 16, 8, 64, torch.float16)
    x, slots = torch.randn(3, 2, 64, device="cuda").half(), torch.arange(3, device="cuda")
    before = c.keys.clone()
    with pytest.raises(ValueError):
        bw.write_cache(x, x, slots, c.keys, c.keys, c.key_meta, c.value_meta, 8, 64)
    with pytest.raises(ValueError):
        bw.write_cache(x, x, slots, c.keys, c.values, c.key_meta, c.key_meta, 8, 64)
    assert torch.equal(c.keys, before)
    bw.read_cache(slots, c.keys, c.keys, c.key_meta, c.key_meta, 8, 64)                 # reading is as good
