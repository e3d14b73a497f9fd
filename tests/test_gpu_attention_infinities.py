"""cache_attention with infinite scores: weight 0 for minus infinity wherever its token lies, NaN where no score is finite."""
import pytest
import torch

from attention_ref import Batch, half_step

pytestmark = pytest.mark.gpu


def _infinite(b, lengths, tokens, head):
    """A batch whose keys of `tokens` (of every sequence that has them) score minus infinity for the queries of `head`; the rows' values stay."""
    at = 0
    b.q[..., 0] = torch.where(b.q[..., 0] < 0, -1.0, 1.0).to(b.dtype)
    share = b.q.shape[1] // b.k.shape[1]
    for s, n in enumerate(lengths):
        b.q[s, head * share:(head + 1) * share, 0] = b.q[s, head * share, 0]
        for t in tokens:
            if t < n:
                b.k[at + t, head, 0] = -float("inf") * b.q[s, head * share, 0].float()
        at += n
    b.cache.write(b.k, b.v, torch.cat(b.slots))


def _expected(b, lengths):
    at, out = 0, []
    kv, dim = b.k.shape[1:]
    for s, n in enumerate(lengths):
        k, v = (x[at:at + n].double().transpose(0, 1) for x in (b.k, b.v))
        at += n
        scores = torch.matmul(b.q[s].double().view(kv, -1, dim), k.transpose(1, 2).contiguous()) * dim ** -0.5
        out.append(torch.matmul(torch.softmax(scores, -1), v.contiguous()).reshape(-1, dim))
    return torch.stack(out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens", [[32], [0], [0, 1, 2], list(range(32, 64)), list(range(16)), list(range(0, 700, 3)), list(range(128, 300)), list(range(40)),
                                    [699, 2999]])
def test_minus_infinity_weighs_nothing_wherever_it_lies(tokens, dim, dtype):
    """33 tokens with the last alone in its wave, whole tiles, whole pieces, and short sequences (one workgroup each, or cut and joined)."""
    for lengths in ([33, 50, 41, 300], [33, 64, 700, 3000, 41]):
        b = Batch(lengths, 8, 2, dim, 16, 16, 64, dtype, seed=len(tokens))
        _infinite(b, lengths, tokens, 1)
        want = _expected(b, lengths)
        got = b.attend().double()
        # (every sequence keeps a finite score, or has none at all and is NaN) the bound of Batch.check without its scores' reach: values below 6
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        kept = ~torch.isnan(want)
        assert bool(((got - want).abs() <= half_step(dtype) * want.abs() + 2.0 ** -13)[kept].all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[1], [33], [600], [5000], [1, 33, 600, 0, 5000]])
def test_no_finite_score_gives_nan_and_no_token_zeros(lengths, dtype):
    b = Batch(lengths, 8, 2, 128, 16, 16, 64, dtype, seed=1)
    _infinite(b, lengths, range(max(lengths)), 0)
    out = b.attend()
    for s, n in enumerate(lengths):
        if n:
            assert torch.isnan(out[s, :4]).all() and torch.isfinite(out[s, 4:]).all()
        else:
            assert not out[s].any()
    b.table[:] = -1                                              # every page outside the cache: no tokens
    assert not b.attend().any()


@pytest.mark.parametrize("at", [0, 31, 32, 599])
def test_plus_infinity_and_infinite_values(at):
    """One score of plus infinity: NaN.  An infinite value under a weight of 0: nothing finite in its channel, and only there."""
    lengths = [33, 600]
    b = Batch(lengths, 8, 2, 128, 16, 16, 64, torch.float16, seed=2)
    b.q[..., 0] = 1
    b.k[33 + at, 1, 0] = float("inf")
    b.cache.write(b.k, b.v, torch.cat(b.slots))
    out = b.attend()
    assert torch.isnan(out[1, 4:]).all() and torch.isfinite(out[1, :4]).all() and torch.isfinite(out[0]).all()
    b.k[33 + at, 1, 0] = -float("inf")
    b.v[33 + at, 1, 7] = float("inf")
    b.cache.write(b.k, b.v, torch.cat(b.slots))
    out = b.attend()
    assert not torch.isfinite(out[1, 4:, 7]).any()
    out[1, 4:, 7] = 0
    assert torch.isfinite(out).all()
