"""cache_attention where the weights of the softmax, or the scales of a head's groups, lie far apart: many small weights beside a large one, groups of one
head that differ by powers of two, scores and scales that rise or fall along the sequence, and values that cancel."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import Batch, half_step, rows

pytestmark = pytest.mark.gpu

FORMATS = [(16, 0, torch.float16), (16, 0, torch.bfloat16), (8, 128, torch.float16), (8, 32, torch.bfloat16), (4, 64, torch.float16), (4, 32, torch.float16)]
CODES = [f for f in FORMATS if f[0] != 16]


def _check(b, out):
    """out against 64 bits, with a bound for every channel from the weights themselves.  With w_t the weights (their sum is 1) and a_t what they multiply
    (|v|; over codes a group's whole range, since code and zero point are multiplied apart):

      half a step of the result's type, and 2^-25 below float16's normal numbers
      2^-22 w_t a_t          a weight as two float16 numbers, each rounded to nearest, or three of bfloat16: 2^-22 and 2^-24
      2^-37 max(w a) a token below float16's normal range: 2^-25, half its smallest step, beside a largest weight of at least 2^12
      2 (dim + 16) 2^-24 reach w_t a_t      scores in float32 (as in Batch.check), and the exponential's argument
      2^-23 (tokens / 32) w_t a_t           float32 sums, one rounding or cut a tile
      2^-18.9 max(w a) a tile               over codes: 32 products cut 2^-16 (8 bits; 4 bits 2^-20) of a unit below the tile's largest
    """
    c = b.cache
    dim, kv = b.q.shape[2], c.keys.shape[1]
    share, scale = b.q.shape[1] // kv, dim ** -0.5
    worst = 0.0
    for s in range(b.q.shape[0]):
        n = len(b.slots[s])
        k, v = (rows(w, m, b.slots[s], b.bits, b.group).transpose(0, 1) for w, m in ((c.keys, c.key_meta), (c.values, c.value_meta)))
        a = v.abs()
        if b.bits != 16:
            pairs = c.value_meta[b.slots[s] // c.page_size, :, :, b.slots[s] % c.page_size].double()
            a = (pairs[..., 0] * (2 ** b.bits - 1)).repeat_interleave(b.group, -1).transpose(0, 1)
        q = b.q[s].double().view(kv, share, dim)
        scores = torch.matmul(k, q.transpose(1, 2).contiguous()) * scale                           # [kv, tokens, share]
        reach = (torch.matmul(k.abs(), q.abs().transpose(1, 2).contiguous()) * scale).amax(1)      # [kv, share]
        weights = torch.softmax(scores, 1)
        for h in range(share):
            w = weights[:, :, h]
            want = (w[..., None] * v).sum(1)
            terms = w[..., None] * a
            total, top = terms.sum(1), terms.amax(1)
            relative = 2.0 ** -22 + 2 * (dim + 16) * 2.0 ** -24 * reach[:, h, None] + 2.0 ** -23 * (n / 32 + 1)
            bound = half_step(b.dtype) * want.abs() + 2.0 ** -25 + relative * total + 2.0 ** -37 * n * top
            if b.bits != 16:
                tiles = torch.nn.functional.pad(terms, (0, 0, 0, -n % 32)).unflatten(1, (-1, 32)).amax(2)
                bound = bound + 2.0 ** -18.9 * tiles.sum(1)
            got = out[s].double().view(kv, share, dim)[:, h]
            worst = max(worst, ((got - want).abs() / bound).max().item())
    assert worst <= 1, f"{worst:.3f} times the bound"


def _filled(b):
    b.cache.write(b.k, b.v, torch.cat(b.slots))
    return b


@pytest.mark.parametrize("gap", [10.0, 12.0, 14.0, 16.0])
@pytest.mark.parametrize("tokens,at", [(8192, 0), (8192, 5000), (65536, 3)])
@pytest.mark.parametrize("bits,group,dtype", FORMATS)
def test_one_token_far_above_many(bits, group, dtype, tokens, at, gap):
    """A token `gap` above the others' scores whose own values are zero: what comes out is the many small weights' part.  Alone, and as 256 sequences
    that share their pages, so that no sequence is cut and the small weights are summed beside the large one."""
    b = Batch([tokens], 4, 2, 128, 64, bits, group or 64, dtype, seed=int(gap), spread=0.5)
    b.q = b.q[:, ::2].repeat_interleave(2, 1)                     # both heads of a key head ask for the same
    q = b.q[0, ::2].float()
    b.k[at] = (q * (gap * 128 ** 0.5 / q.pow(2).sum(-1, keepdim=True))).to(dtype)
    b.v.fill_(1.0)
    b.v[at] = 0
    _filled(b)
    out = b.attend()
    b.check(out)
    _check(b, out)
    many = b.cache.attend(b.q.expand(256, -1, -1), b.table.expand(256, -1), b.lengths.expand(256))
    for s in (0, 100, 255):
        b.check(many[s:s + 1])
        _check(b, many[s:s + 1])


@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("heads", [8, 16, 32])
@pytest.mark.parametrize("bits,group,dtype", CODES)
def test_groups_of_one_head_of_very_different_size(bits, group, dtype, heads, first):
    """Values of the groups of a head 2^8 ... 2^-8: every group as exact as if it were alone, whichever is the largest."""
    if group == 128:
        pytest.skip("one group")
    b = Batch([4000] * 12, heads, 2, 128, 32, bits, group, dtype, seed=heads)
    sizes = 2.0 ** torch.linspace(8, -8, 128 // group, device="cuda").repeat_interleave(group)
    b.v = (b.v.float() * (sizes.flip(0) if first else sizes)).to(dtype)
    b.q = (b.q.float() * 2.5).to(dtype)
    _filled(b)
    out = b.attend()
    b.check(out)
    _check(b, out)


@pytest.mark.parametrize("heads", [4, 10, 32])
@pytest.mark.parametrize("scores", [-40.0, 0.0, 40.0])
@pytest.mark.parametrize("sizes", [-16.0, 0.0, 16.0])
@pytest.mark.parametrize("bits,group,dtype", FORMATS)
def test_scores_and_values_that_rise_or_fall(bits, group, dtype, sizes, scores, heads):
    """Along the sequence scores go from 0 to `scores` and values from 2^(-sizes/2) to 2^(sizes/2), every other group the other way round."""
    if bits == 16 and sizes:
        sizes /= 2                                               # (values of float16 itself)
    n = 3000
    b = Batch([n, 77], heads, 2, 128, 64, bits, group or 64, dtype, seed=heads, spread=0.5)
    way = torch.arange(n, device="cuda") / n
    share = heads // 2
    b.q = b.q[:, ::share].repeat_interleave(share, 1)
    q = b.q[0, ::share].float()
    b.k[:n] = (b.k[:n].float() + way[:, None, None] * (q * (scores * 128 ** 0.5 / q.pow(2).sum(-1, keepdim=True)))[None]).to(dtype)
    sign = 1 - 2 * (torch.arange(128, device="cuda") // (group or 64) % 2)
    b.v[:n] = (b.v[:n].float() * 2.0 ** (sizes * (way[:, None] - 0.5) * sign)[:, None]).to(dtype)
    _filled(b)
    _check(b, b.attend())


@pytest.mark.parametrize("bits,group", [(8, 32), (4, 64)])
def test_scales_at_both_ends_of_float16(bits, group):
    """A group whose scales are float16's smallest beside one with its largest, in every other token the other way round, with equal scores."""
    cache = bw.PagedCache(8, 1, 128, 64, bits, group, torch.bfloat16)
    slots = torch.arange(512, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(4)
    cache.values.random_(-2 ** 31, 2 ** 31 - 1, generator=gen)
    cache.key_meta.fill_(1.0)
    ends = torch.tensor([2.0 ** -24, 65504.0], device="cuda").half()
    which = (torch.arange(64, device="cuda")[None] + torch.arange(128 // group, device="cuda")[:, None]) % 2
    which[-1] = 0                                                # and one group of the smallest alone
    cache.value_meta[..., 0] = ends[which]
    cache.value_meta[..., 1] = 3
    q = torch.zeros(1, 4, 128, device="cuda", dtype=torch.bfloat16)
    out = cache.attend(q, torch.arange(8, dtype=torch.int32, device="cuda")[None], torch.tensor([512], dtype=torch.int32, device="cuda"))[0].double()
    v = rows(cache.values, cache.value_meta, slots, bits, group)[:, 0]
    a = (cache.value_meta[..., 0].double() * (2 ** bits - 1)).transpose(2, 3).reshape(512, -1).repeat_interleave(group, -1)
    bound = half_step(torch.bfloat16) * v.mean(0).abs() + (2.0 ** -22 + 2.0 ** -18.9 + 2.0 ** -19) * a.amax(0) + 2.0 ** -37 * a.amax(0)
    worst = ((out - v.mean(0)).abs() / bound).max().item()
    assert worst <= 1, f"{worst:.3f} times the bound"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_cancel(dtype):
    """Weights of a few tokens that are nearly the same and values 1 and -1: what comes out is the difference of float32 weights.  A score is one product
    (exact in float32); scaling, exponent, exponential, sums and the quotient are at most 16 float32 operations on a weight and one for every token."""
    lengths = [2, 3, 4, 5, 6, 7, 8] * 20
    b = Batch(lengths, 16, 4, 64, 16, 16, 64, dtype, seed=5)
    b.k[..., 1:] = 0
    b.k[..., 0] = torch.rand(b.k.shape[:2], device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(dtype)
    b.v = torch.where(b.v > 0.5, 1.0, -1.0).to(dtype)
    _filled(b)
    out = b.attend()
    at = 0
    worst = 0.0
    for s, n in enumerate(lengths):
        k, v = b.k[at:at + n].double(), b.v[at:at + n].double()
        at += n
        scores = b.q[s].double()[:, 0].view(4, 4, 1) * k[..., 0].t()[:, None] * 64 ** -0.5
        want = torch.matmul(torch.softmax(scores, -1), v.transpose(0, 1).contiguous()).view(16, 64)
        bound = half_step(dtype) * want.abs() + (16 + n) * 2.0 ** -24 + 2.0 ** -25
        worst = max(worst, ((out[s].double() - want).abs() / bound).max().item())
    assert worst <= 1, f"{worst:.3f} times the bound"


@pytest.mark.parametrize("tokens", [2, 40, 700])
@pytest.mark.parametrize("gap", [20.0, 24.0, 27.0, 30.0, 40.0])
def test_values_at_the_upper_end_of_bfloat16(gap, tokens):
    """Values up to 2^127 under one weight near 1 among small ones: finite, as products of float32 weights are.  The token far above is the last, so that
    its score is met after the others' (2^(gap / ln 2) lower)."""
    b = Batch([tokens, tokens], 8, 2, 128, 32, 16, 64, torch.bfloat16, seed=int(gap), spread=0.02)
    b.q = b.q[:, ::4].repeat_interleave(4, 1)
    for s in range(2):
        q = b.q[s, ::4].float()
        for step in range(5):                                    # several raised scores, a fifth of the gap apart
            at = (s + 1) * tokens - 1 - 16 * step
            if at >= s * tokens:
                b.k[at] = (q * ((gap - step * gap / 5) * 128 ** 0.5 / q.pow(2).sum(-1, keepdim=True))).bfloat16()
    b.v = (b.v.float().clamp(-1.9, 1.9) * 2.0 ** 127).bfloat16()
    _filled(b)
    out = b.attend().double()
    for s in range(2):
        k, v = (x[s * tokens:(s + 1) * tokens].double().transpose(0, 1) for x in (b.k, b.v))
        w = torch.softmax(torch.matmul(b.q[s].double().view(2, 4, 128), k.transpose(1, 2).contiguous()) * 128 ** -0.5, -1)
        want = torch.matmul(w, v.contiguous()).reshape(8, 128)
        # scores in float32: 2 (dim + 16) 2^-24 of at most gap + 1, of values below 2^128
        assert torch.isfinite(out[s]).all()
        assert bool(((out[s] - want).abs() <= half_step(torch.bfloat16) * want.abs() + 2 * 144 * 2.0 ** -24 * (gap + 1) * 2.0 ** 128).all())


@pytest.mark.parametrize("bits,group,dtype", FORMATS)
@pytest.mark.parametrize("heads", [2, 12, 32])
def test_one_token_gives_its_values(heads, bits, group, dtype):
    """A weight of 1 is exact: a sequence of one token gives what the cache holds, rounded once, whatever its score."""
    b = Batch([1] * 70, heads, 2, 128, 16, bits, group or 64, dtype, seed=heads, spread=3.0)
    c = b.cache
    want = rows(c.values, c.value_meta, torch.cat(b.slots), bits, b.group).to(dtype).repeat_interleave(heads // 2, 1)
    assert torch.equal(b.attend(), want)


@pytest.mark.parametrize("bits,group,dtype", FORMATS)
def test_one_token_above_all_gives_its_values(bits, group, dtype):
    """So does the only token with a weight, wherever it lies: the others' scores are 2000 lower."""
    for at in (0, 33, 299):
        b = Batch([300, 700], 4, 2, 128, 16, bits, group or 64, dtype, seed=at)
        b.q.fill_(1.0)
        b.k[:300].fill_(-177.0)
        b.k[at].fill_(1.0)
        _filled(b)
        want = rows(b.cache.values, b.cache.value_meta, b.slots[0][at:at + 1], bits, b.group).to(dtype).repeat_interleave(2, 1)
        assert torch.equal(b.attend()[0], want[0])
