"""C entry points of rotation, cache and attention with sizes that they refuse: status codes and workspace sizes, without a GPU."""
import pytest

from bitween_amd.kernels import hip_loader

OK, EINVAL, EUNSUPPORTED, EALIGN = 0, -1, -2, -3
P = 4096                                                         # stands for a device address: never followed on the host


def _heads(**other):
    fields = dict(tokens=4, q_heads=2, k_heads=1, dim=64, rotary=64, cos=P, sin=P, table_rows=10, positions=P, q_weight=P, k_weight=None, weight_dtype=0, eps=1e-6)
    return hip_loader.Heads(**{**fields, **other})


@pytest.mark.parametrize("fields", [dict(dim=264), dict(dim=2048), dict(dim=4096), dict(dim=65536), dict(dim=1 << 30), dict(dim=60, rotary=40), dict(rotary=60), dict(tokens=1 << 40),
                                    dict(tokens=(1 << 63) - 1), dict(q_heads=70000), dict(k_heads=(1 << 31) - 1), dict(weight_dtype=3), dict(cos=P + 4)])
def test_no_workspace_for_a_gradient_that_is_refused(fields):
    lib, h = hip_loader.load(), _heads(**fields)
    assert lib.bw_rotate_heads_grad_workspace_bytes(h) == 0
    assert lib.bw_rotate_heads_grad(h, 0, P, 128, 64, P, 64, 64, P, 128, 64, None, 0, 0, P, P, P, None, P, 1 << 30, None) in (EUNSUPPORTED, EALIGN)


@pytest.mark.parametrize("fields", [dict(), dict(weight_dtype=1), dict(weight_dtype=2), dict(k_weight=P), dict(q_weight=None, k_weight=P), dict(dim=256), dict(dim=8, rotary=8)])
def test_a_workspace_for_a_gradient_that_is_taken(fields):
    h = _heads(**fields)
    assert hip_loader.load().bw_rotate_heads_grad_workspace_bytes(h) >= 2 * h.dim * 4          # a row of each kind at least


def _cache(**other):
    fields = dict(keys=P, values=P, key_meta=P, value_meta=P, pages=4, kv_heads=2, page_size=16, dim=64, bits=8, group=32, dtype=0)
    return hip_loader.Cache(**{**fields, **other})


@pytest.mark.parametrize("page_size", [16, 1024])
@pytest.mark.parametrize("power", [53, 54, 55, 58, 59, 60, 61, 62])
def test_tables_whose_tokens_pass_64_bits_are_refused(power, page_size):
    """2^54 pages of 1024 tokens are 2^64: a table without room, if the product wraps."""
    lib, c = hip_loader.load(), _cache(page_size=page_size)
    for extra in (0, 1):
        assert lib.bw_cache_attention(c, 0, P, 1, 2, 128, 64, P, (1 << power) + extra, 4, P, 1.0, P, P, 1 << 30, None) == EUNSUPPORTED
        assert lib.bw_cache_attention_workspace_bytes(c, 1, 2, (1 << power) + extra) == 0


def test_caches_whose_values_pass_63_bits_are_refused():
    """(2^31 - 1) pages of 1024 rows, 65535 heads of 256 values: two such tensors share memory wherever they lie, if their size wraps to nothing they do not."""
    lib, c = hip_loader.load(), _cache(pages=(1 << 31) - 1, page_size=1024, kv_heads=65535, dim=256, values=2 * P, value_meta=3 * P)
    assert lib.bw_cache_write(c, 0, 1, P, 16776960, 256, P, 16776960, 256, P, None) == EUNSUPPORTED
    assert lib.bw_cache_read(c, 0, 1, P, P, P, None) == EUNSUPPORTED
    assert lib.bw_cache_attention_workspace_bytes(c, 1, 65535, 4) == 0


@pytest.mark.parametrize("dim,rotary", [(80, 40), (40, 40), (136, 136), (24, 8), (64, 64), (256, 256)])
def test_rotations_are_refused_from_2_31_heads_and_2_36_values_on(dim, rotary):
    """Whatever lanes a head has: the limits that the header states, for the forward and its gradient (refused here by their pointers' alignment instead)."""
    lib = hip_loader.load()
    tokens = min((1 << 31) - 1, ((1 << 36) - 1) // dim) // 3     # of 3 heads

    def status(tokens):
        h = _heads(tokens=tokens, dim=dim, rotary=rotary, cos=P + 4)
        return lib.bw_rotate_heads(h, 0, P, 3 * dim, dim, P, 3 * dim, dim, P, P, None), lib.bw_rotate_heads_grad(
            h, 0, P, 3 * dim, dim, P, 3 * dim, dim, P, 3 * dim, dim, None, 0, 0, P, P, None, None, None, 0, None)

    assert status(tokens) == (EALIGN, EALIGN)
    assert status(tokens + 1) == (EUNSUPPORTED, EUNSUPPORTED)
