"""cache_attention against 64 bits: formats, heads, lengths, pages, and what lies where nothing may look."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import Batch, rows

pytestmark = pytest.mark.gpu

FORMATS = [(16, 0, torch.float16), (16, 0, torch.bfloat16), (8, 32, torch.float16), (8, 64, torch.bfloat16), (8, 128, torch.float16), (4, 32, torch.bfloat16),
           (4, 64, torch.float16), (4, 128, torch.bfloat16), (4, 128, torch.float16)]


@pytest.mark.parametrize("bits,group,dtype", FORMATS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 128), (32, 8, 128), (12, 12, 64), (64, 4, 128), (20, 1, 256), (40, 2, 128), (5, 1, 64), (6, 2, 96), (2, 2, 192)])
def test_formats_and_heads(heads, kv_heads, dim, bits, group, dtype):
    if group and dim % group:
        pytest.skip("the group does not divide this head")
    b = Batch([1, 2, 15, 16, 17, 31, 33, 0, 64, 65, 127, 128, 129, 300, 511, 1000], heads, kv_heads, dim, 16, bits, group or 64, dtype, seed=heads)
    b.check(b.attend())


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 72, 80, 120, 136, 200, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_odd_heads_at_16_bits(dim, dtype):
    b = Batch([3, 50, 0, 257, 1], 6, 3, dim, 32, 16, 64, dtype, seed=dim)
    b.check(b.attend())


@pytest.mark.parametrize("bits,dtype", [(8, torch.bfloat16), (4, torch.float16)])
@pytest.mark.parametrize("share", [3, 7, 12])
@pytest.mark.parametrize("group,groups", [(32, n) for n in range(1, 9)] + [(64, n) for n in range(1, 5)] + [(128, 1), (128, 2)])
def test_every_number_of_groups_with_few_and_many_queries(group, groups, share, bits, dtype):
    b = Batch([1, 20, 33, 0, 450, 1300], 2 * share, 2, group * groups, 32, bits, group, dtype, seed=group + groups)
    b.check(b.attend())
    b = Batch([70, 511], 2 * share, 2, group * groups, 64, bits, group, dtype, seed=groups)
    b.check(b.attend())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("bits,group,dtype", [(16, 0, torch.float16), (8, 64, torch.float16), (4, 32, torch.bfloat16)])
def test_pages(page, bits, group, dtype):
    b = Batch([page - 1, page, page + 1, 3 * page + 5, 1, 700], 8, 2, 64, page, bits, group or 64, dtype, seed=page)
    b.check(b.attend())


@pytest.mark.parametrize("lengths", [[1], [2000], [0], [0, 0, 0], [12345], [0, 30000], [1] * 300, [40] * 257, [5000, 1, 1, 1, 1, 1, 1, 3], list(range(130))])
@pytest.mark.parametrize("bits,group", [(16, 0), (8, 128), (4, 64)])
def test_lengths(lengths, bits, group):
    b = Batch(lengths, 4, 2, 128, 64, bits, group or 64, torch.float16, seed=len(lengths))
    b.check(b.attend())


@pytest.mark.parametrize("room", [513, 1000, 1024, 1025])
@pytest.mark.parametrize("bits,group,dtype", [(16, 0, torch.float16), (8, 128, torch.bfloat16), (4, 64, torch.float16)])
def test_many_sequences_with_room_for_about_1024(room, bits, group, dtype):
    b = Batch([room] + [(37 * i) % 1000 for i in range(35)], 8, 4, 128, 16, bits, group or 64, dtype, seed=room)
    b.check(b.attend())
    b = Batch([5, room, 0, 200], 8, 4, 128, 16, bits, group or 64, dtype, seed=room + 1)
    b.check(b.attend())


@pytest.mark.parametrize("bits,group,dtype", [(16, 0, torch.bfloat16), (4, 128, torch.float16), (8, 64, torch.float16)])
def test_one_long_sequence(bits, group, dtype):
    b = Batch([100003], 32, 8, 128, 64, bits, group or 64, dtype, seed=1)
    b.check(b.attend())


def test_wide_table_short_sequences_and_table_rows_apart():
    """A table with room for far more than the sequences hold, whose rows are a slice of a wider one."""
    b = Batch([3, 100, 0, 17], 8, 8, 128, 16, 16, 64, torch.float16, width=4096)
    wide = torch.full((4, 5000), -7, dtype=torch.int32, device="cuda")
    wide[:, 3:4099] = b.table
    b.table = wide[:, 3:4099]
    b.check(b.attend())


def test_lengths_outside_the_table_and_pages_outside_the_cache():
    b = Batch([64, 64, 64, 64], 8, 2, 64, 16, 16, 64, torch.float16)
    b.lengths.copy_(torch.tensor([2 ** 31 - 1, -5, -2 ** 31, 65], dtype=torch.int32))
    b.check(b.attend(), lengths=[64, 0, 0, 64])                  # cut to the table
    b = Batch([64, 64, 40], 8, 2, 64, 16, 8, 64, torch.float16)
    b.table[0, 1], b.table[1], b.table[2, 2] = -1, 2 ** 31 - 1, b.cache.keys.shape[0]
    b.slots = [torch.cat([b.slots[0][:16], b.slots[0][32:]]), b.slots[1][:0], b.slots[2][:32]]
    b.check(b.attend())                                          # pages without tokens


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64), (4, 128)])
def test_what_lies_behind_the_last_token_does_not_matter(bits, group):
    b = Batch([5, 16, 37, 0], 8, 4, 128, 16, bits, group or 64, torch.float16)
    want = b.attend()
    for fill in (float("inf"), float("-inf"), 65504.0, -65504.0, 0.0):
        c = b.cache
        kept = b.k, b.v, torch.cat(b.slots)
        for t in (c.keys, c.values) if bits == 16 else (c.key_meta, c.value_meta):
            t.fill_(fill)
        c.write(*kept)
        assert torch.equal(b.attend(), want)


@pytest.mark.parametrize("bits,group,dtype", [(16, 0, torch.float16), (16, 0, torch.bfloat16), (8, 64, torch.bfloat16), (4, 32, torch.float16)])
def test_scores_far_apart_and_far_from_zero(bits, group, dtype):
    """One token takes all the weight, wherever it lies; scores of hundreds; a scale of its own, a negative one, and 0."""
    for at in (0, 31, 700, 1499):
        b = Batch([1500], 4, 2, 128, 64, bits, group or 64, dtype, seed=at, spread=4.0)
        b.k[at] = b.q[0].view(2, 2, 128)[:, 0] * 8
        b.cache.write(b.k, b.v, b.slots[0])
        b.check(b.attend())
    for scale in (0.0, 1.0, -0.3):
        b.check(b.attend(scale), scale)


@pytest.mark.parametrize("bits,group", [(8, 64), (4, 128)])
def test_values_of_very_different_size(bits, group):
    """Every other token has values 2^19 times larger and a score some 60 lower (e^-60 2^19 is nothing): the small ones are not lost beside
    them, whichever come first."""
    for big in (0, 1):
        b = Batch([200], 4, 2, 128, 16, bits, group, torch.float16, seed=big)
        small = (torch.arange(200, device="cuda") % 2 == big)[:, None, None]
        b.v = torch.where(small, b.v * 2.0 ** -12, b.v * 2.0 ** 7)
        b.k = torch.where(small, b.k, -6 * b.q[0].view(2, 2, 128).sum(1))
        b.cache.write(b.k, b.v, b.slots[0])
        got = b.attend()[0].double()
        k, v = (rows(w, m, b.slots[0], bits, group).transpose(0, 1).contiguous() for w, m in ((b.cache.keys, b.cache.key_meta), (b.cache.values, b.cache.value_meta)))
        scores = torch.matmul(b.q[0].double().view(2, 2, 128), k.transpose(1, 2).contiguous()) * 128 ** -0.5
        want = torch.matmul(torch.softmax(scores, -1), v).reshape(4, 128)
        top = v[:, small[:, 0, 0]].abs().amax()
        assert want.abs().max() <= top                            # the large ones have no part in it
        assert bool(((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -14 * top + 2.0 ** -25).all())


def test_infinities_and_nan_in_cached_rows():
    """An infinite value leaves nothing finite where it enters (its channel of the heads that read it), a NaN key in the whole heads that read it."""
    b = Batch([50, 50], 4, 2, 64, 16, 16, 64, torch.float16)
    b.v[7, 0, 5] = float("inf")
    b.cache.write(b.k, b.v, torch.cat(b.slots))
    out = b.attend()
    assert not torch.isfinite(out[0, :2, 5]).any() and torch.isfinite(out[0, 2:]).all() and torch.isfinite(out[1]).all()
    assert torch.isfinite(out[0, :2, torch.arange(64, device="cuda") != 5]).all()
    b.v[7, 0, 5] = 0
    b.k[60, 1, 3] = float("nan")
    b.cache.write(b.k, b.v, torch.cat(b.slots))
    out = b.attend()
    assert torch.isnan(out[1, 2:]).all() and torch.isfinite(out[1, :2]).all() and torch.isfinite(out[0]).all()


def test_queries_as_parts_of_a_projection_and_types_of_the_table():
    b = Batch([70, 3, 129], 8, 2, 64, 16, 16, 64, torch.bfloat16)
    want = b.attend()
    fused = torch.randn(3, 12, 64, device="cuda").bfloat16()
    fused[:, :8] = b.q
    q = b.q
    for view in (fused[:, :8], q.transpose(0, 1).contiguous().transpose(0, 1), torch.empty(3, 8, 65, device="cuda", dtype=torch.bfloat16)[..., :64].copy_(q),
                 q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(b.cache.attend(view, b.table, b.lengths), want)
    assert torch.equal(b.cache.attend(q, b.table.long(), b.lengths.long()), want)
    assert torch.equal(b.cache.attend(q, b.table.t().contiguous().t(), b.lengths), want)
    assert b.cache.attend(q[:0], b.table[:0], b.lengths[:0]).shape == (0, 8, 64)
    shared = b.table[:1].expand(3, -1)                           # three sequences over the same pages
    out = b.cache.attend(q[:1].expand(3, 8, 64), shared, b.lengths[:1].expand(3))
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2]) and torch.equal(out[0], want[0])


@pytest.mark.parametrize("bits,group", [(16, 0), (4, 64)])
def test_the_same_bits_every_time_and_on_another_stream(bits, group):
    b = Batch([9000, 1, 4000, 70], 16, 4, 128, 64, bits, group or 64, torch.float16)
    want = b.attend()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        assert torch.equal(b.attend(), want)
        with torch.cuda.stream(side):
            other = b.attend()
        here = b.attend()                                        # at the same time
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, want) and torch.equal(here, want)


def test_captured_calls_follow_lengths_and_table_and_two_graphs_stay_apart():
    b = Batch([3000, 500, 1], 8, 2, 128, 16, 16, 64, torch.float16)
    b.attend()
    torch.cuda.synchronize()
    graphs, outs, queries = [], [], [b.q.clone(), b.q.clone()]
    for q in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(b.cache.attend(q, b.table, b.lengths))
        graphs.append(graph)
    full = b.lengths.clone()
    for seed in range(4):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        n = [int(torch.randint(0, int(m) + 1, (1,), generator=torch.Generator().manual_seed(seed + i))) for i, m in enumerate(full)]
        b.lengths.copy_(torch.tensor(n, dtype=torch.int32))
        for q in queries:
            q.copy_(torch.randn(q.shape, device="cuda", generator=gen))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for q, out in zip(queries, outs):
            assert torch.equal(out, b.cache.attend(q, b.table, b.lengths))
            b.q = q
            b.check(out, lengths=n)


@pytest.mark.parametrize("bits,group,dtype", [(16, 0, torch.bfloat16), (8, 64, torch.float16), (4, 128, torch.float16)])
def test_a_decode_loop(bits, group, dtype):
    """A prompt and twenty single tokens: rotation, write and attention as a decoder calls them, each token against the rows written before."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    batch, heads, kv, dim, page = 3, 8, 2, 128, 16
    cache = bw.PagedCache(40, kv, dim, page, bits, group or 64, dtype)
    table = torch.randperm(40, device="cuda", generator=gen)[:12].view(3, 4).int()
    angle = torch.arange(64, device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(64, device="cuda", dtype=torch.float64) / 64)
    cos, sin = angle.cos().float(), angle.sin().float()
    start = [20, 1, 33]
    lengths = torch.tensor(start, dtype=torch.int32, device="cuda")
    holder = Batch(start, heads, kv, dim, page, bits, group or 64, dtype)
    holder.cache, holder.table, holder.lengths = cache, table, lengths
    seq = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(start)])
    pos = torch.cat([torch.arange(n, device="cuda") for n in start])
    qkv = torch.randn(len(pos), heads + 2 * kv, dim, device="cuda", generator=gen).to(dtype)
    _, k = bw.rotate_heads(qkv[:, :heads], qkv[:, heads:heads + kv], cos, sin, pos)
    cache.write(k, qkv[:, heads + kv:], cache.slots(table, pos, seq))
    for _ in range(20):
        qkv = torch.randn(batch, heads + 2 * kv, dim, device="cuda", generator=gen).to(dtype)
        pos = lengths.long()
        q, k = bw.rotate_heads(qkv[:, :heads], qkv[:, heads:heads + kv], cos, sin, pos)
        cache.write(k, qkv[:, heads + kv:], cache.slots(table, pos))
        lengths += 1
        out = cache.attend(q, table, lengths)
        holder.q = q
        holder.slots = [cache.slots(table, torch.arange(int(n), device="cuda"), torch.full((int(n),), b, device="cuda")) for b, n in enumerate(lengths)]
        holder.check(out)


@pytest.mark.parametrize("bits,group", [(8, 64), (4, 128)])
@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** 118, 2.0 ** 121, 2.0 ** -100, 2.0 ** -130])
def test_queries_at_the_ends_of_bfloat16(size, bits, group):
    """Over codes the queries' exponent is taken out and put back into the scores: at the upper end one token has all the weight (scores 2^90 and
    more apart), at the lower end every token has the same."""
    b = Batch([70, 700], 4, 2, 128, 32, bits, group, torch.bfloat16, seed=3)
    b.q = (b.q.float() * size).to(torch.bfloat16)
    b.check(b.attend())


@pytest.mark.parametrize("bits,group,dtype", [(16, 0, torch.float16), (8, 64, torch.bfloat16), (4, 32, torch.float16)])
def test_a_padded_step_is_the_step_of_its_sequences(bits, group, dtype):
    """Rotation, write and attention of a batch whose idle rows have position -1, length 0 and a table of anything, captured once and replayed: the
    sequences get what they get alone, idle rows zeros, and the cache nothing of theirs."""
    heads, kv, dim, page = 8, 2, 128, 32
    gen = torch.Generator(device="cuda").manual_seed(bits)
    caches = [bw.PagedCache(12, kv, dim, page, bits, group or 64, dtype) for _ in range(2)]
    angle = torch.arange(100, device="cuda", dtype=torch.float32)[:, None] / 10000.0 ** (torch.arange(64, device="cuda", dtype=torch.float32) / 64)
    cos, sin = angle.cos(), angle.sin()
    table = torch.tensor([[3, 1, 9], [0, 0, 0], [7, 4, 2], [-5, 2 ** 30, 3]], dtype=torch.int32, device="cuda")
    active = torch.tensor([0, 2], device="cuda")
    lengths, positions = torch.tensor([31, 0, 64, 0], dtype=torch.int32, device="cuda"), torch.tensor([30, -1, 63, -1], device="cuda")
    for b in (0, 2):
        n = int(positions[b])
        x = torch.randn(n, 2 * kv, dim, device="cuda", generator=gen).to(dtype)
        for cache in caches:
            cache.write(x[:, :kv], x[:, kv:], cache.slots(table, torch.arange(n, device="cuda"), torch.full((n,), b, device="cuda")))
    qkv = torch.zeros(4, heads + 2 * kv, dim, device="cuda", dtype=dtype)

    def step(cache, qkv, positions, table, lengths):
        q, k = bw.rotate_heads(qkv[:, :heads], qkv[:, heads:heads + kv], cos, sin, positions)
        cache.write(k, qkv[:, heads + kv:], cache.slots(table, positions))
        return cache.attend(q, table, lengths)

    step(caches[0], qkv, positions, table, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], qkv, positions, table, lengths)
    for _ in range(4):
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=gen))
        qkv[1::2] = float("nan")
        graph.replay()
        want = step(caches[1], qkv[active], positions[active], table[active], lengths[active])
        assert torch.equal(out[active], want) and not out[1::2].any()
        for a, b in zip((getattr(c, name) for c in caches[:1] for name in ("keys", "values", "key_meta", "value_meta")),
                        (getattr(c, name) for c in caches[1:] for name in ("keys", "values", "key_meta", "value_meta"))):
            assert a is None and b is None or torch.equal(a, b)
        positions += (positions >= 0).long()
        lengths += (lengths > 0).int()


def test_wide_whole_numbers_outside_stay_outside():
    """int64 tables and lengths: what does not fit 32 bits must not come back as a page or a length that does."""
    b = Batch([64, 64, 5], 8, 2, 64, 16, 16, 64, torch.float16)
    table, lengths = b.table.long(), b.lengths.long()
    table[0, 2:] = 2 ** 32 + table[0, 2:]
    table[1, :] -= 2 ** 33
    lengths[1] += 2 ** 32
    out = b.cache.attend(b.q, table, lengths)
    b.check(out, lengths=[32, 0, 5])
    full = b.cache.attend(b.q, b.table, torch.tensor([2 ** 32 + 1, 64, -2 ** 32 + 5], device="cuda"))
    b.check(full, lengths=[64, 64, 0])


@pytest.mark.parametrize("bits,group,pages", [(16, 0, 66000), (8, 64, 132000), (4, 128, 264000)])
def test_pages_behind_four_gibibytes(bits, group, pages):
    """8.6 GB of keys, so that every other page lies behind 32 bits of bytes (and behind 31 bits of values)."""
    b = Batch([1000, 70, 0, 300], 8, 8, 128, 64, bits, group or 64, torch.float16, spare=pages)
    page_bytes = b.cache.keys[0].nbytes
    assert int(b.table[b.table < 2 ** 30].max()) * page_bytes > 2 ** 32
    b.check(b.attend())
