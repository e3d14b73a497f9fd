"""How many workgroups the prompt attention and its gradients take, without a GPU."""
import pytest

from test_attention_entry_points import EUNSUPPORTED, P
from test_prompt_entry_points import EWORKSPACE, _backward, _forward, _prompt

MANY = [dict(q_tokens=1 << 17, k_tokens=1 << 17, sequences=1 << 17, q_heads=64, kv_heads=64, dim=8), dict(q_tokens=1 << 18, k_tokens=1 << 18, sequences=1 << 18, q_heads=63, kv_heads=63, dim=8),
        dict(q_tokens=200000, k_tokens=200000, sequences=200000, q_starts=P, k_starts=P, q_heads=64, kv_heads=64, dim=8),
        dict(q_tokens=100000, k_tokens=10 ** 8, sequences=100000, q_starts=P, k_starts=P, q_heads=16, kv_heads=16, dim=8)]


@pytest.mark.parametrize("fields", MANY)
def test_the_gradients_take_what_the_forward_takes(fields):
    """As far as the workspace, which is not there: nothing is launched."""
    row = fields["q_heads"] * 8
    rows = {f"{name}_row": row for name in ("q", "grad", "k", "v")}
    heads = {f"{name}_head": 8 for name in ("q", "grad", "k", "v")}
    assert _backward(_prompt(**fields), ws=None, size=0, **rows, **heads) == EWORKSPACE


def test_more_workgroups_than_there_may_be():
    p = _prompt(q_tokens=10, k_tokens=10, sequences=1 << 20, q_starts=P, k_starts=P, q_heads=4096, kv_heads=4096, dim=8)
    rows = dict(q_row=32768, k_row=32768, v_row=32768, q_head=8, k_head=8, v_head=8)
    assert _forward(p, ws=None, size=0, **rows) == EUNSUPPORTED
    assert _backward(p, ws=None, size=0, grad_row=32768, grad_head=8, **rows) == EUNSUPPORTED
