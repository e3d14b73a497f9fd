"""Refusals of rotate_heads, the cache and cache_attention that need no GPU: status codes of the C entry points before anything is launched, and the
Python layer's errors."""
import ctypes

import pytest
import torch

import bitween_amd as bw
from bitween_amd.kernels import hip_loader
from bitween_amd.kernels.hip_loader import BitweenHipError

OK, EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = 0, -1, -2, -3, -5
P = 4096                                                         # stands for a device address: never followed on the host


def _cache(**other):
    fields = dict(keys=P, values=P, key_meta=P, value_meta=P, pages=4, kv_heads=2, page_size=16, dim=64, bits=8, group=32, dtype=0)
    return hip_loader.Cache(**{**fields, **other})


CACHES = [(dict(keys=None), EINVAL), (dict(values=None), EINVAL), (dict(key_meta=None), EINVAL), (dict(value_meta=None), EINVAL), (dict(pages=0), EINVAL),
          (dict(kv_heads=0), EINVAL), (dict(page_size=0), EINVAL), (dict(dim=0), EINVAL), (dict(bits=3), EINVAL), (dict(bits=2), EUNSUPPORTED),
          (dict(group=0), EINVAL), (dict(group=48), EINVAL), (dict(group=16), EUNSUPPORTED), (dict(bits=16, dtype=2), EUNSUPPORTED),
          (dict(bits=16, dim=68), EUNSUPPORTED), (dict(bits=16, dim=264), EUNSUPPORTED), (dict(page_size=8), EUNSUPPORTED), (dict(page_size=48), EUNSUPPORTED),
          (dict(page_size=2048), EUNSUPPORTED), (dict(pages=1 << 31), EUNSUPPORTED), (dict(keys=P + 8), EALIGN), (dict(value_meta=P + 4), EALIGN)]


@pytest.mark.parametrize("fields,status", CACHES)
def test_caches_that_are_refused(fields, status):
    lib, c = hip_loader.load(), _cache(**fields)
    assert lib.bw_cache_write(c, 0, 1, P, 128, 64, P, 128, 64, P, None) == status
    assert lib.bw_cache_read(c, 0, 1, P, P, P, None) == status
    assert lib.bw_cache_attention(c, 0, P, 1, 2, 128, 64, P, 4, 4, P, 1.0, P, P, 1 << 30, None) == status
    assert lib.bw_cache_attention_workspace_bytes(c, 1, 2, 4) == 0


def test_cache_entry_points_check_their_arguments():
    lib, c, c16 = hip_loader.load(), _cache(), _cache(bits=16, dtype=1)
    assert lib.bw_cache_write(None, 0, 1, P, 128, 64, P, 128, 64, P, None) == EINVAL
    assert lib.bw_cache_write(c, 0, 0, None, 0, 0, None, 0, 0, None, None) == OK
    for hole in (3, 6, 9):
        args = [c, 0, 1, P, 128, 64, P, 128, 64, P, None]
        args[hole] = None
        assert lib.bw_cache_write(*args) == EINVAL
    assert lib.bw_cache_write(c, 0, -1, P, 128, 64, P, 128, 64, P, None) == EINVAL
    assert lib.bw_cache_write(c, 2, 1, P, 128, 64, P, 128, 64, P, None) == EUNSUPPORTED
    assert lib.bw_cache_write(c16, 0, 1, P, 128, 64, P, 128, 64, P, None) == EUNSUPPORTED           # float16 rows into a bfloat16 cache
    for at, value in ((3, P + 2), (4, 129), (5, 60), (6, P + 8), (7, 4), (8, 2), (9, P + 4)):
        args = [c, 0, 1, P, 128, 64, P, 128, 64, P, None]
        args[at] = value
        assert lib.bw_cache_write(*args) == EALIGN
    assert lib.bw_cache_read(c, 0, 0, None, None, None, None) == OK
    assert lib.bw_cache_read(c, 0, 1, None, P, P, None) == EINVAL
    assert lib.bw_cache_read(c, 2, 1, P, P, P, None) == EUNSUPPORTED and lib.bw_cache_read(c16, 0, 1, P, P, P, None) == EUNSUPPORTED
    assert lib.bw_cache_read(c, 0, 1, P, P + 2, P, None) == EALIGN


def test_keys_and_values_that_share_memory_are_not_written():
    lib = hip_loader.load()
    size = 4 * 2 * 16 * 64                                       # bytes of keys or values at 8 bits
    for fields in (dict(), dict(values=P + size), dict(values=P + size - 16, value_meta=P + size), dict(values=P - size + 16, value_meta=P + size),
                   dict(values=P + size, value_meta=P + size // 32 * 4 - 16), dict(bits=16, values=P + 2 * size - 16)):
        assert lib.bw_cache_write(_cache(**fields), 0, 1, P, 128, 64, P, 128, 64, P, None) == EINVAL


def test_attention_entry_point_checks_its_arguments():
    lib, c, c16 = hip_loader.load(), _cache(), _cache(bits=16, dtype=1)
    ok = [c, 0, P, 1, 2, 128, 64, P, 4, 4, P, 1.0, P, P, 1 << 30, None]

    def call(**other):
        names = ["cache", "act", "q", "B", "heads", "q_row", "q_head", "table", "max_pages", "table_row", "lengths", "scale", "out", "ws", "ws_bytes", "stream"]
        args = list(ok)
        for name, value in other.items():
            args[names.index(name)] = value
        return lib.bw_cache_attention(*args)

    assert call(B=0, q=None, table=None, lengths=None, out=None) == OK
    for name in ("q", "table", "lengths", "out"):
        assert call(**{name: None}) == EINVAL
    assert call(B=-1) == EINVAL and call(heads=0) == EINVAL and call(heads=3) == EINVAL and call(max_pages=0) == EINVAL
    assert call(B=2, table_row=3) == EINVAL
    assert call(act=2) == EUNSUPPORTED and call(cache=c16) == EUNSUPPORTED
    assert call(B=1 << 40) == EUNSUPPORTED and call(max_pages=1 << 40) == EUNSUPPORTED
    assert call(q=P + 2) == EALIGN and call(out=P + 8) == EALIGN and call(q_row=100) == EALIGN and call(table=P + 2) == EALIGN


def test_rotation_entry_points_check_their_arguments():
    lib = hip_loader.load()

    def heads(**other):
        fields = dict(tokens=4, q_heads=2, k_heads=1, dim=64, rotary=64, cos=P, sin=P, table_rows=10, positions=P, q_weight=P, k_weight=None, weight_dtype=0, eps=1e-6)
        return hip_loader.Heads(**{**fields, **other})

    def forward(h, act=0, q=P, row=128, out=P):
        return lib.bw_rotate_heads(h, act, q, row, 64, P, 64, 64, out, P, None)

    def backward(h, act=0, x=P, gw=P, ws=P, size=1 << 30, out=P, row=128):
        return lib.bw_rotate_heads_grad(h, act, P, row, 64, P, 64, 64, x, 128, 64, None, 0, 0, out, P, gw, None, ws, size, None)

    for call in (forward, backward):
        assert call(None) == EINVAL
        for field in ("tokens", "q_heads", "k_heads", "dim", "rotary", "table_rows"):
            assert call(heads(**{field: -1})) == EINVAL
        for field in ("cos", "sin", "positions"):
            assert call(heads(**{field: None})) == EINVAL
        assert call(heads(rotary=72)) == EINVAL
        assert call(heads(), act=2) == EUNSUPPORTED and call(heads(weight_dtype=1)) == EUNSUPPORTED
        for fields in (dict(dim=68, rotary=64), dict(rotary=60), dict(dim=264), dict(tokens=1 << 40), dict(q_heads=70000), dict(tokens=1 << 29),
                       dict(tokens=1 << 31)):
            assert call(heads(**fields)) == EUNSUPPORTED
        assert call(heads(cos=P + 4)) == EALIGN and call(heads(positions=P + 4)) == EALIGN and call(heads(q_weight=P + 2)) == EALIGN
        assert call(heads(), out=None) == EINVAL and call(heads(), out=P + 2) == EALIGN and call(heads(), row=100) == EALIGN
    assert forward(heads(tokens=0), q=None) == OK and forward(heads(), q=None) == EINVAL and forward(heads(), q=P + 2) == EALIGN
    assert backward(heads(), x=None) == EINVAL                   # a weight needs the forward's input
    assert backward(heads(q_weight=None)) == EINVAL              # a gradient of no weight
    assert backward(heads(), ws=None, size=0) == EWORKSPACE and backward(heads(), size=100) == EWORKSPACE and backward(heads(), ws=P + 4) == EALIGN
    assert lib.bw_rotate_heads_grad_workspace_bytes(heads(q_weight=None)) == 0 and lib.bw_rotate_heads_grad_workspace_bytes(heads()) > 0
    assert lib.bw_rotate_heads_grad_workspace_bytes(None) == 0


def test_constructor():
    c = bw.PagedCache(3, 2, 128, 32, bits=4, group_size=64, device="cpu")
    assert c.keys.shape == c.values.shape == (3, 2, 32, 16) and c.keys.dtype == torch.int32
    assert c.key_meta.shape == c.value_meta.shape == (3, 2, 2, 32, 2) and c.key_meta.dtype == torch.float16
    c = bw.PagedCache(3, 2, 80, 16, dtype=torch.bfloat16, device="cpu")
    assert c.keys.shape == (3, 2, 16, 80) and c.keys.dtype == torch.bfloat16 and c.key_meta is None and c.page_size == 16
    table = torch.tensor([[2, 0], [1, 1]], dtype=torch.int32)
    assert c.slots(table, torch.tensor([17, 3])).tolist() == [1, 19]
    assert c.slots(table, torch.tensor([0, 16, 5]), torch.tensor([0, 0, 1])).tolist() == [32, 0, 21]
    for other, error in ((dict(bits=3), ValueError), (dict(bits=2), NotImplementedError), (dict(dtype=torch.float32), TypeError), (dict(pages=0), ValueError),
                         (dict(page_size=24), NotImplementedError), (dict(page_size=8), NotImplementedError), (dict(head_dim=100), NotImplementedError),
                         (dict(head_dim=512), NotImplementedError), (dict(bits=8, group_size=48), ValueError), (dict(bits=8, group_size=16), NotImplementedError),
                         (dict(bits=4, head_dim=80, group_size=32), ValueError)):
        with pytest.raises(error):
            bw.PagedCache(**{**dict(pages=2, kv_heads=2, head_dim=64, page_size=16, device="cpu"), **other})


def test_errors_of_the_python_layer():
    """Wrong types and shapes raise what the package raises elsewhere; CPU tensors raise BitweenHipError, there is no CPU path."""
    half = dict(dtype=torch.float16)
    q, k, cos, pos = torch.zeros(3, 4, 64, **half), torch.zeros(3, 2, 64, **half), torch.ones(10, 32), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(BitweenHipError):
        bw.rotate_heads(q, k, cos, cos, pos)
    with pytest.raises(TypeError):
        bw.rotate_heads(q.float(), k, cos, cos, pos)
    with pytest.raises(TypeError):
        bw.rotate_heads(q, k.bfloat16(), cos, cos, pos)
    with pytest.raises(TypeError):
        bw.rotate_heads(q, None, cos, cos, pos)
    c = bw.PagedCache(4, 2, 64, 16, device="cpu")
    slots, table, lengths = torch.arange(3), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for call in (lambda: c.write(k, k, slots), lambda: c.read(slots), lambda: c.attend(q, table, lengths)):
        with pytest.raises(BitweenHipError):
            call()
    with pytest.raises(NotImplementedError):
        bw.read_cache(slots, c.keys, c.values, bits=2)
    with pytest.raises(ValueError):
        bw.read_cache(slots, c.keys, c.values, bits=5)
    with pytest.raises(TypeError):
        bw.read_cache(slots, c.keys, c.values, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        bw.cache_attention(q, table, lengths, c.keys, c.values, bits=8)
    with pytest.raises(ValueError):
        bw.cache_attention(q, table, lengths, c.keys, c.values, c.keys, c.values)
    eight = bw.PagedCache(4, 2, 64, 16, bits=8, group_size=32, device="cpu")
    with pytest.raises(ValueError):
        bw.write_cache(k, k, slots, eight.keys, eight.values, eight.key_meta, eight.value_meta, 8, 64)
    with pytest.raises(ValueError):
        bw.write_cache(k, k, slots, eight.keys, eight.values, eight.key_meta, eight.value_meta, 8, 48)
    with pytest.raises(TypeError):
        bw.write_cache(k, k, slots, eight.keys, eight.values, None, None, 8, 32)


@pytest.mark.gpu
def test_errors_on_the_gpu():
    half = dict(dtype=torch.float16, device="cuda")
    q, k, cos, pos = torch.zeros(3, 4, 64, **half), torch.zeros(3, 2, 64, **half), torch.ones(10, 32, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for error, args in ((ValueError, (q, k[:2], cos, cos, pos)), (ValueError, (q, k[..., :56], cos, cos, pos)), (ValueError, (q, k, cos, cos[:5], pos)),
                        (ValueError, (q, k, torch.ones(10, 40, device="cuda"), torch.ones(10, 40, device="cuda"), pos)), (TypeError, (q, k, cos, cos, pos.float())),
                        (TypeError, (q, k, cos.long(), cos, pos)), (ValueError, (q, k, cos, cos, pos, torch.ones(63, **half))), (BitweenHipError, (q, k, cos.cpu(), cos, pos)),
                        (TypeError, (q, k, cos, cos, pos, torch.ones(64, device="cuda", dtype=torch.bfloat16))),
                        (ValueError, (q, k, cos, cos, pos, torch.ones(64, **half), torch.ones(64, device="cuda"))),
                        (NotImplementedError, (q, k, cos[:, :30].contiguous(), cos[:, :30].contiguous(), pos)),
                        (NotImplementedError, (q, k, cos.clone().requires_grad_(True), cos, pos)),
                        (NotImplementedError, (torch.zeros(3, 1, 512, **half), torch.zeros(3, 1, 512, **half), cos, cos, pos))):
        with pytest.raises(error):
            bw.rotate_heads(*args)
    c = bw.PagedCache(4, 2, 64, 16)
    slots, table, lengths = torch.arange(3, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for error, call in ((ValueError, lambda: c.write(k, k, slots[:2])), (ValueError, lambda: c.write(q, q, slots)), (TypeError, lambda: c.write(k.bfloat16(), k.bfloat16(), slots)),
                        (TypeError, lambda: c.write(k, k, slots.float())), (BitweenHipError, lambda: c.write(k, k, slots.cpu())),
                        (BitweenHipError, lambda: c.write(k.clone().requires_grad_(True), k, slots)), (ValueError, lambda: c.read(slots[None])),
                        (ValueError, lambda: c.attend(q[:, :3], table, lengths)), (ValueError, lambda: c.attend(q, table[:2], lengths)),
                        (ValueError, lambda: c.attend(q, table, lengths[:2])), (TypeError, lambda: c.attend(q.bfloat16(), table, lengths)),
                        (TypeError, lambda: c.attend(q, table.float(), lengths)), (BitweenHipError, lambda: c.attend(q.clone().requires_grad_(True), table, lengths)),
                        (ValueError, lambda: bw.cache_attention(q, table, lengths, c.keys[::2], c.values[::2])),
                        (NotImplementedError, lambda: bw.cache_attention(torch.zeros(3, 4, 4, **half), table, lengths, c.keys[..., :4].contiguous(), c.values[..., :4].contiguous()))):
        with pytest.raises(error):
            call()
    with torch.no_grad():
        c.attend(q.clone().requires_grad_(True), table, lengths)


def test_slots_of_positions_without_a_page_are_padding():
    c = bw.PagedCache(3, 2, 128, 16, device="cpu")
    table = torch.tensor([[2, 0], [-1, 3], [1, 1]], dtype=torch.int32)
    assert c.slots(table, torch.tensor([-1, 3, 32])).tolist() == [-1, -1, -1]
    assert c.slots(table, torch.tensor([31, 16, 5, 17, 31], dtype=torch.int32), torch.tensor([0, 1, 2, 2, 0])).tolist() == [15, -1, 21, 17, 15]
    with pytest.raises(ValueError):
        c.slots(table, torch.tensor([1]))


def test_what_is_no_tensor_is_named():
    t = torch.zeros(1)
    with pytest.raises(TypeError):
        bw.read_cache(t, None, None)
    with pytest.raises(TypeError):
        bw.read_cache(t, None, None, bits=8)
    with pytest.raises(TypeError):
        bw.cache_attention(None, t, t, None, None)
    with pytest.raises(TypeError):
        bw.cache_attention(t, t, t, None, None)
    with pytest.raises(TypeError):
        bw.write_cache(None, None, None, None, None)
    with pytest.raises(TypeError):
        bw.rotate_heads(None, None, None, None, None)
