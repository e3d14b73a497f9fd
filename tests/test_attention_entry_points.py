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
