"""cache_attention with a window and sinks: against 64 bits over the tokens that count, in every format of the cache."""
import pytest
import torch

import bitween_amd as bw
from attention_ref import Batch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


class Windowed(Batch):
    """A batch of which only some tokens count: check() goes by them, and the table's entries of pages that hold none of them are numbers far outside."""

    def limit(self, window, sinks):
        size = self.cache.page_size
        for b, slots in enumerate(self.slots):
            n = len(slots)
            at = torch.arange(n, device="cuda")
            keep = (at >= n - window) | (at < sinks)
            gone = torch.ones(self.table.shape[1], dtype=torch.bool, device="cuda")
            gone[(at[keep] // size).unique()] = False
            self.table[b, gone] = -(2 ** 30) + b
            # a token that does not count may be anything
            out = slots[~keep]
            page, row = out // size, out % size
            if self.bits == 16:
                self.cache.keys[page, :, row], self.cache.values[page, :, row] = float("nan"), float("inf")
            else:
                self.cache.key_meta[page, :, :, row], self.cache.value_meta[page, :, :, row] = float("nan"), float("inf")
            self.slots[b] = slots[keep]
        return self


CASES = [  # lengths, query heads, key heads, dim, page, window, sinks
    ([1, 2, 31, 32, 33, 0], 4, 2, 64, 16, 1, 0), ([100, 7, 0, 513], 8, 2, 128, 16, 33, 5), ([2000], 8, 8, 128, 64, 100, 4), ([65, 64, 63, 200], 4, 1, 64, 32, 64, 64), ([3000, 17, 900], 16, 1, 128, 16, 1000, 1),
    ([300, 301, 302, 303, 304, 305], 5, 1, 96, 128, 47, 16), ([5000, 4999], 4, 4, 256, 16, 4000, 31), ([700] * 70, 2, 2, 64, 16, 130, 33), ([10000], 32, 8, 128, 64, 256, 2000),
    ([1024, 1, 40], 40, 2, 64, 1024, 500, 100), ([90, 1500], 4, 2, 64, 16, 2, 1), ([256], 1, 1, 128, 16, 16, 240)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits,group", [(16, 0), (8, 32), (8, 64), (4, 32), (4, 64)])
@pytest.mark.parametrize("case", CASES)
def test_against_64_bits(case, bits, group, dtype):
    lengths, heads, kv, dim, page, window, sinks = case
    if bits != 16 and dim % group:
        pytest.skip("groups do not divide the head")
    batch = Windowed(lengths, heads, kv, dim, page, bits, group, dtype, seed=sum(lengths)).limit(window, sinks)
    out = batch.cache.attend(batch.q, batch.table, batch.lengths, window=window, sinks=sinks)
    batch.check(out)
    assert torch.equal(out, batch.cache.attend(batch.q, batch.table, batch.lengths, window=window, sinks=sinks))


@pytest.mark.parametrize("bits,group,dim", [(16, 0, 80), (8, 128, 128), (4, 128, 256), (16, 0, 200)])
def test_heads_of_other_sizes(bits, group, dim):
    batch = Windowed([1200, 3, 77], 6, 3, dim, 32, bits, group, torch.float16).limit(70, 9)
    batch.check(batch.cache.attend(batch.q, batch.table, batch.lengths, window=70, sinks=9))


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64), (4, 32)])
def test_a_window_of_everything_is_none(bits, group):
    batch = Batch([900, 33, 0, 1, 400], 8, 2, 64, 16, bits, group, torch.float16)
    want = batch.attend()
    for window, sinks in ((None, 7), (2 ** 40, 0), (100000, 5), (912, 0), (912, 2 ** 40)):
        assert torch.equal(batch.cache.attend(batch.q, batch.table, batch.lengths, window=window, sinks=sinks), want)
    # sinks that meet the window leave nothing out either
    got = batch.cache.attend(batch.q, batch.table, batch.lengths, window=500, sinks=400)
    batch.check(got)


def test_pages_outside_and_lengths_that_change_under_a_capture():
    batch = Windowed([600, 600, 600], 4, 2, 64, 16, 16, 0, torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = batch.cache.attend(batch.q, batch.table, batch.lengths, window=50, sinks=3)
    for n in (600, 51, 50, 1, 0, 333, 600):
        batch.lengths[1] = n
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, batch.cache.attend(batch.q, batch.table, batch.lengths, window=50, sinks=3))
        torch.cuda.synchronize()
    # a page of the window outside the cache is one without tokens, and nothing at all is zeros
    batch.table[2] = -1
    got = batch.cache.attend(batch.q, batch.table, batch.lengths, window=50, sinks=3)
    assert not got[2].any() and got[0].any()
    batch.table[2, 0] = 2 ** 31 - 1
    assert not batch.cache.attend(batch.q, batch.table, batch.lengths, window=50, sinks=3)[2].any()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = batch.cache.attend(batch.q, batch.table, batch.lengths, window=50, sinks=3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, got)


def test_half_a_tile_without_pages():
    """The window begins in the second half of a tile whose first half has a page in the table that is none of the sequence's, and whose second half has none at all: no token counts."""
    batch = Windowed([64], 2, 1, 64, 16, 16, 0, torch.float16)
    batch.table[0, 3] = -1
    assert not batch.cache.attend(batch.q, batch.table, batch.lengths, window=16).any()


def test_refusals():
    batch = Batch([40], 4, 2, 64, 16, 16, 0, torch.float16)
    for kw, error in ((dict(window=0), ValueError), (dict(window=-3), ValueError), (dict(window=5, sinks=-1), ValueError), (dict(window=2.0), TypeError), (dict(window=True), TypeError),
                      (dict(window=5, sinks=None), TypeError)):
        with pytest.raises(error):
            batch.cache.attend(batch.q, batch.table, batch.lengths, **kw)
