"""What autograd is told by the cache and its attention, which have no derivatives: refusals instead of results without their part of a graph."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import bitween_amd as bw
from bitween_amd.kernels.hip_loader import BitweenHipError

pytestmark = pytest.mark.gpu


def _calls(bits, slots_type=torch.int64, table_type=torch.int32):
    """name -> (inputs that may take part in a graph, call of a list of them).  The types decide whether a call is taken as it is or converted first."""
    dtype = torch.bfloat16
    c = bw.PagedCache(4, 2, 64, 16, bits, 64, dtype)
    x = torch.randn(3, 2, 64, device="cuda").to(dtype)
    q = torch.randn(3, 4, 64, device="cuda").to(dtype)
    slots, table, lengths = (torch.arange(3, device="cuda", dtype=slots_type), torch.zeros(3, 2, dtype=table_type, device="cuda"),
                             torch.ones(3, dtype=table_type, device="cuda"))
    cache = [t for t in (c.keys, c.values, c.key_meta, c.value_meta) if t is not None]

    def held(tensors):
        return (*tensors, None, None)[:4] + (bits, 64)

    return {"write": ([x, x.clone(), *cache], lambda t: bw.write_cache(t[0], t[1], slots, *held(t[2:]))),
            "read": (cache, lambda t: bw.read_cache(slots, *held(t), dtype=dtype)),
            "attend": ([q, *cache], lambda t: bw.cache_attention(t[0], table, lengths, *held(t[1:])))}


@pytest.mark.parametrize("name", ["write", "read", "attend"])
@pytest.mark.parametrize("converted", [False, True])
@pytest.mark.parametrize("bits", [16, 8])
def test_forward_mode_is_refused(bits, converted, name):
    types = (torch.int32, torch.int64) if converted else (torch.int64, torch.int32)
    inputs, call = _calls(bits, *types)[name]
    call(inputs)
    for i, t in enumerate(inputs):
        if not t.is_floating_point():
            continue
        with fwad.dual_level():
            dual = [fwad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(inputs)]
            for context in (torch.enable_grad(), torch.no_grad()):
                with context, pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(dual)
            call(inputs)                                          # within a level, without a tangent


@pytest.mark.parametrize("converted", [False, True])
def test_forward_mode_of_the_rotation_s_tables_is_refused(converted):
    q, cos = torch.randn(3, 4, 64, device="cuda").half(), torch.rand(5, 32, device="cuda")
    positions = torch.arange(3, device="cuda", dtype=torch.int32 if converted else torch.int64)
    with fwad.dual_level():
        dual = fwad.make_dual(cos, torch.ones_like(cos))
        for tables in ((dual, cos), (cos, dual)):
            for context in (torch.enable_grad(), torch.no_grad()):
                with context, pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    bw.rotate_heads(q, q, *tables, positions)


@pytest.mark.parametrize("name", ["write", "read", "attend"])
@pytest.mark.parametrize("converted", [False, True])
@pytest.mark.parametrize("bits", [16, 8])
def test_tensors_that_ask_for_gradients_are_refused(bits, converted, name):
    """Queries, new rows, 16-bit keys and values, scales: with grad mode a call that would leave their gradients out raises, without it the call is made."""
    types = (torch.int32, torch.int64) if converted else (torch.int64, torch.int32)
    inputs, call = _calls(bits, *types)[name]
    want = call(inputs)
    for i, t in enumerate(inputs):
        if not t.is_floating_point():
            continue
        asking = [x.detach().requires_grad_(True) if j == i else x for j, x in enumerate(inputs)]
        with pytest.raises(BitweenHipError, match="no gradient"):
            call(asking)
        with torch.no_grad():
            got = call(asking)
        for a, b in zip(*((x if isinstance(x, tuple) else (x,)) for x in (got, want))):
            assert a is None and b is None or torch.equal(a, b)
