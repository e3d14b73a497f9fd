"""append_cache with norms over heads that hold an infinity or a NaN."""
import pytest
import torch

import bitween_amd as bw
from test_gpu_append import _cache, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dim,rotary", [(128, 64), (64, 64), (32, 32), (40, 40)])
def test_a_normed_head_with_an_infinity(dim, rotary, bits, dtype):
    """x * rsqrt(mean(x^2) + eps) * weight of a head with an infinity: the root's inverse is 0, NaN where x is infinite (and at the value that turns with it), zeros elsewhere, as in the two
    calls; of a head with a NaN nothing but NaN.  Other heads and tokens are as they are without."""
    if bits != 16 and dim % 32:
        pytest.skip("groups of 32")
    (q, k, v, cos, sin, positions), w = _inputs(20, 2, 2, dim, rotary, dtype, weights=True)
    clean, slots = _cache(2, dim, bits, 32, 16, dtype, 20)
    q, k = q.clone(), k.clone()
    want_q = clean.append(q, k, v, cos, sin, positions, slots, *w)
    want_k, _ = clean.read(slots)
    q[2, 0, 3], k[3, 1, 5], k[7, 0, dim - 1], q[9, 1, 1] = float("inf"), float("inf"), float("-inf"), float("nan")
    cache, slots = _cache(2, dim, bits, 32, 16, dtype, 20)
    got = cache.append(q, k, v, cos, sin, positions, slots, *w)
    keys, _ = cache.read(slots)
    two_q, two_k = bw.rotate_heads(q, k, cos, sin, positions, *w)
    plain, _ = _cache(2, dim, bits, 32, 16, dtype, 20)
    plain.write(two_k, v, slots)
    written, _ = plain.read(slots)
    for x, two, before, heads in ((got, two_q, want_q, ((2, 0), (9, 1))), (keys, written, want_k, ((3, 1), (7, 0)))):
        for token, head in heads:
            assert torch.equal(x[token, head].nan_to_num(nan=-7.0), two[token, head].nan_to_num(nan=-7.0)), (token, head)
            x[token, head] = before[token, head]
        assert torch.equal(x, before)
    assert torch.isnan(two_q[2, 0]).sum() == 2 and torch.isnan(two_q[9, 1]).all() and (two_q[2, 0].nan_to_num(nan=0.0) == 0).all()
