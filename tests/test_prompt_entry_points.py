"""C entry points of several axes, append, windows and prompts with what they refuse: status codes and workspace sizes, without a GPU; errors of the Python layer; registers."""
import pytest
import torch

import bitween_amd as bw
from bitween_amd.kernels import hip_loader
from test_abi_and_host import _kernel_metadata
from test_attention_entry_points import EALIGN, EINVAL, EUNSUPPORTED, OK, P, _cache, _heads

EWORKSPACE = -5
BIG = 1 << 40



def _axes(*sections, interleaved=0, count=None):
    return hip_loader.Axes(len(sections) if count is None else count, (hip_loader.ctypes.c_int * 4)(*sections[:4]), interleaved)


@pytest.mark.parametrize("axes", [None, _axes(), _axes(32, count=5), _axes(32, count=-1), _axes(16, 15), _axes(16, 17), _axes(40, -8), _axes(8, 16, 8, interleaved=1),
                                  _axes(0, 32, interleaved=1)])
def test_axes_that_do_not_fit_the_pairs_are_refused(axes):
    lib, h, c = hip_loader.load(), _heads(q_weight=None), _cache(kv_heads=1)
    assert lib.bw_rotate_axes(h, axes, 0, P, 128, 64, P, 64, 64, P, P, None) == EINVAL
    assert lib.bw_rotate_axes_grad(h, axes, 0, P, 128, 64, P, 64, 64, None, 0, 0, None, 0, 0, P, P, None, None, None, 0, None) == EINVAL
    if axes is not None:                                         # (none at all is one position)
        assert lib.bw_cache_append(c, h, axes, 0, P, 128, 64, P, 64, 64, P, 64, 64, P, P, None) == EINVAL


def test_axes_that_fit_go_on_to_the_other_checks():
    lib = hip_loader.load()
    for axes in (_axes(32), _axes(0, 32), _axes(16, 8, 8), _axes(8, 8, 8, 8), _axes(12, 10, 10, interleaved=1), _axes(11, 11, 10, interleaved=1), _axes(16, 16, interleaved=1)):
        assert lib.bw_rotate_axes(_heads(cos=P + 4), axes, 0, P, 128, 64, P, 64, 64, P, P, None) == EALIGN
        assert lib.bw_rotate_axes(_heads(tokens=0), axes, 0, None, 128, 64, None, 64, 64, None, None, None) == OK
        assert lib.bw_rotate_axes(_heads(), axes, 2, P, 128, 64, P, 64, 64, P, P, None) == EUNSUPPORTED
        assert lib.bw_rotate_axes(_heads(tokens=1 << 40), axes, 0, P, 128, 64, P, 64, 64, P, P, None) == EUNSUPPORTED
    assert lib.bw_rotate_axes(None, _axes(32), 0, P, 128, 64, P, 64, 64, P, P, None) == EINVAL


def test_append_checks_its_arguments():
    lib = hip_loader.load()

    def call(cache=_cache(kv_heads=1), heads=_heads(), act=0, **other):
        a = dict(q=P, q_row=128, k=P, k_row=64, v=P, v_row=64, slots=P, out=P)
        a.update(other)
        return lib.bw_cache_append(cache, heads, None, act, a["q"], a["q_row"], 64, a["k"], a["k_row"], 64, a["v"], a["v_row"], 64, a["slots"], a["out"], None)

    shared = dict(kv_heads=1)
    far = dict(kv_heads=1, values=P << 20, value_meta=P << 22, key_meta=P << 21)
    assert call(heads=_heads(tokens=0), q=None, k=None, v=None, slots=None, out=None) == OK
    for name in ("q", "k", "v", "slots", "out"):
        assert call(_cache(**far), **{name: None}) == EINVAL
    assert call(None) == EINVAL and call(heads=None) == EINVAL
    assert call(_cache(**shared)) == EINVAL                      # keys and values share memory
    assert call(_cache(**dict(far, kv_heads=2))) == EINVAL       # of other heads than the cache
    assert call(_cache(**dict(far, dim=128))) == EINVAL
    assert call(_cache(**far), act=2) == EUNSUPPORTED
    assert call(_cache(**dict(far, bits=16, dtype=1))) == EUNSUPPORTED
    for heads in (dict(tokens=1 << 40), dict(q_heads=70000), dict(tokens=1 << 29, q_weight=None)):
        assert call(_cache(**far), _heads(**heads)) == EUNSUPPORTED
    for other in (dict(q=P + 2), dict(k=P + 8), dict(v=P + 2), dict(out=P + 8), dict(slots=P + 4), dict(q_row=100), dict(v_row=65)):
        assert call(_cache(**far), **other) == EALIGN


def test_a_window_checks_its_arguments():
    lib, c = hip_loader.load(), _cache()

    def call(window=5, sinks=1, **other):
        a = dict(q=P, B=1, heads=2, row=128, table=P, pages=4, lengths=P, out=P, ws=P, size=1 << 30, act=0)
        a.update(other)
        return lib.bw_cache_attention_window(c, a["act"], a["q"], a["B"], a["heads"], a["row"], 64, a["table"], a["pages"], 4, a["lengths"], 1.0, window, sinks, a["out"], a["ws"], a["size"],
                                             None)

    assert call(B=0, q=None, table=None, lengths=None, out=None) == OK
    assert call(window=-1) == EINVAL and call(sinks=-1) == EINVAL
    for name in ("q", "table", "lengths", "out"):
        assert call(**{name: None}) == EINVAL
    assert call(act=2) == EUNSUPPORTED and call(pages=1 << 54) == EUNSUPPORTED and call(B=1 << 40) == EUNSUPPORTED
    assert call(q=P + 2) == EALIGN and call(row=100) == EALIGN


@pytest.mark.parametrize("sinks", [0, 4, 1 << 62, (1 << 63) - 1])
@pytest.mark.parametrize("window", [0, 1, 4096, 1 << 62, (1 << 63) - 1])
def test_workspaces_of_windows(window, sinks):
    """No larger than that of the whole table, whatever the numbers; none for a table that is refused."""
    lib, c = hip_loader.load(), _cache(bits=16)
    whole = lib.bw_cache_attention_workspace_bytes(c, 1, 2, 10000)
    assert 0 <= lib.bw_cache_attention_window_workspace_bytes(c, 1, 2, 10000, window, sinks) <= whole
    assert lib.bw_cache_attention_window_workspace_bytes(c, 1, 2, 1 << 60, window, sinks) == 0
    assert lib.bw_cache_attention_window_workspace_bytes(c, 1, 2, 10000, -1, 0) == 0


def _prompt(**other):
    fields = dict(q_tokens=10, k_tokens=20, q_starts=None, k_starts=None, sequences=1, q_heads=4, kv_heads=2, dim=64, window=0, sinks=0, scale=0.125)
    return hip_loader.Prompt(**{**fields, **other})


def _forward(p, act=0, **other):
    a = dict(q=P, q_row=256, q_head=64, k=P, k_row=128, k_head=64, v=P, v_row=128, v_head=64, out=P, lse=P, ws=P, size=1 << 40)
    a.update(other)
    return hip_loader.load().bw_prompt_attention(p, act, a["q"], a["q_row"], a["q_head"], a["k"], a["k_row"], a["k_head"], a["v"], a["v_row"], a["v_head"], a["out"], a["lse"],
                                                 a["ws"], a["size"], None)


def _backward(p, act=0, **other):
    a = dict(grad=P, grad_row=256, grad_head=64, q=P, q_row=256, q_head=64, k=P, k_row=128, k_head=64, v=P, v_row=128, v_head=64, out=P, lse=P, gq=P, gk=P, gv=P, ws=P, size=1 << 40)
    a.update(other)
    return hip_loader.load().bw_prompt_attention_grad(p, act, a["grad"], a["grad_row"], a["grad_head"], a["q"], a["q_row"], a["q_head"], a["k"], a["k_row"], a["k_head"], a["v"],
                                                      a["v_row"], a["v_head"], a["out"], a["lse"], a["gq"], a["gk"], a["gv"], a["ws"], a["size"], None)


WRONG = [(dict(q_tokens=-1), EINVAL), (dict(k_tokens=-1), EINVAL), (dict(sequences=0), EINVAL), (dict(q_heads=0), EINVAL), (dict(kv_heads=0), EINVAL), (dict(kv_heads=3), EINVAL),
         (dict(dim=0), EINVAL), (dict(window=-1), EINVAL), (dict(sinks=-1), EINVAL), (dict(q_starts=P), EINVAL), (dict(k_starts=P), EINVAL), (dict(sequences=3), EINVAL),
         (dict(dim=60), EUNSUPPORTED), (dict(dim=264), EUNSUPPORTED), (dict(q_heads=131072, kv_heads=65536), EUNSUPPORTED), (dict(q_tokens=BIG), EUNSUPPORTED),
         (dict(k_tokens=BIG), EUNSUPPORTED), (dict(q_tokens=1 << 29), EUNSUPPORTED), (dict(k_tokens=1 << 30), EUNSUPPORTED), (dict(q_tokens=(1 << 63) - 1, k_tokens=(1 << 63) - 1), EUNSUPPORTED),
         (dict(q_starts=P, k_starts=P, sequences=(1 << 31) - 1), EUNSUPPORTED), (dict(q_starts=P + 2, k_starts=P), EALIGN), (dict(q_starts=P, k_starts=P + 1), EALIGN)]


@pytest.mark.parametrize("fields,status", WRONG)
def test_prompts_that_are_refused(fields, status):
    lib, p = hip_loader.load(), _prompt(**fields)
    assert _forward(p) == status and _backward(p) == status
    assert lib.bw_prompt_attention_workspace_bytes(p) == 0 and lib.bw_prompt_attention_grad_workspace_bytes(p) == 0


def test_prompt_entry_points_check_their_arguments():
    p = _prompt()
    for call in (_forward, _backward):
        assert call(None) == EINVAL and call(p, act=2) == EUNSUPPORTED and call(p, act=-1) == EUNSUPPORTED
        for name in ("q", "k", "v", "out"):
            assert call(p, **{name: None}) == EINVAL
            assert call(p, **{name: P + 8}) == EALIGN
        for name in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head"):
            assert call(p, **{name: 100}) == EALIGN
        for name in ("k_row", "v_row"):
            assert call(p, **{name: 1 << 24}) == EUNSUPPORTED and call(p, **{name: -128}) == EUNSUPPORTED
    assert _forward(_prompt(q_tokens=0), q=None, out=None, k=None, v=None) == OK
    assert _backward(_prompt(q_tokens=0, k_tokens=0), grad=None, q=None, k=None, v=None, out=None, lse=None, gq=None, gk=None, gv=None) == OK
    assert _backward(p, grad=None) == EINVAL and _backward(p, lse=None) == EINVAL and _backward(p, grad=P + 2) == EALIGN
    for name in ("gq", "gk", "gv"):
        assert _backward(p, **{name: P + 8}) == EALIGN
    for name in ("q_row", "grad_row"):
        assert _backward(p, **{name: 1 << 24}) == EUNSUPPORTED and _backward(p, **{name: -256}) == EUNSUPPORTED
    for name in ("q_head", "grad_head"):
        assert _backward(p, **{name: 1 << 30}) == EUNSUPPORTED and _backward(p, **{name: -64}) == EUNSUPPORTED
    assert _backward(_prompt(q_heads=64), q_head=1 << 27) == EUNSUPPORTED
    assert _backward(p, ws=None, size=0) == EWORKSPACE and _backward(p, size=8) == EWORKSPACE and _backward(p, ws=P + 4) == EALIGN
    few = _prompt(q_tokens=1, k_tokens=30000)                    # one row, a long axis: in parts
    size = hip_loader.load().bw_prompt_attention_workspace_bytes(few)
    assert size > 0
    assert _forward(few, ws=None, size=0) == EWORKSPACE and _forward(few, size=size - 1) == EWORKSPACE and _forward(few, ws=P + 4) == EALIGN


def test_workspaces_of_prompts():
    lib = hip_loader.load()
    assert lib.bw_prompt_attention_workspace_bytes(None) == 0 and lib.bw_prompt_attention_grad_workspace_bytes(None) == 0
    assert lib.bw_prompt_attention_workspace_bytes(_prompt(q_tokens=8192, k_tokens=8192, q_heads=32, kv_heads=8)) == 0           # enough rows: no parts
    for fields in (dict(q_tokens=1, k_tokens=100000), dict(q_tokens=63, k_tokens=32063, q_heads=32, kv_heads=8, dim=128), dict(q_tokens=64, k_tokens=64000, sequences=64),
                   dict(q_tokens=64, k_tokens=64000, sequences=64, q_starts=P, k_starts=P)):
        p = _prompt(**fields)
        size = lib.bw_prompt_attention_workspace_bytes(p)
        row = p.q_tokens * p.q_heads * (p.dim + 2) * 4
        assert size % row == 0 and size <= 64 * row              # a reference, a sum and the values of each part
        assert lib.bw_prompt_attention_workspace_bytes(_prompt(**fields, window=16)) <= size
        for large in (p.k_tokens, 1 << 40, 1 << 62, (1 << 63) - 1):
            for sinks in (0, large):
                assert lib.bw_prompt_attention_workspace_bytes(_prompt(**fields, window=large, sinks=sinks)) == size         # a window of everything is none
        assert lib.bw_prompt_attention_grad_workspace_bytes(p) >= p.q_tokens * p.q_heads * 4


def test_errors_of_the_python_layer():
    half = torch.zeros(4, 2, 64, dtype=torch.float16)
    table, at = torch.zeros(10, 32), torch.arange(4)
    error, pages = hip_loader.BitweenHipError, [torch.zeros(1, 2, 16, 64, dtype=torch.float16) for _ in range(2)]
    with pytest.raises(error):
        bw.prompt_attention(half, half, half)
    with pytest.raises(error):
        bw.rotate_heads(half, half, table, table, at[None].expand(2, 4), sections=(16, 16))
    with pytest.raises(error):
        bw.append_cache(half, half, half, table, table, at, at, *pages)
    for what in (None, 3, [1.0]):
        with pytest.raises(TypeError):
            bw.prompt_attention(what, half, half)


def test_prompt_and_window_kernels_keep_their_values_in_registers():
    """Up to heads of 128 the forward and the queries' gradient keep everything in registers, the keys' gradient all but a few words that its loop does not touch; of 256 two
    hundred bytes of a lane lie in memory."""
    kernels = list(_kernel_metadata(hip_loader.library_path()))
    rows = [k for k in kernels if "prompt_forward" in k[".name"]]
    grads = [k for k in kernels if "prompt_query_grad" in k[".name"] or "prompt_key_grad" in k[".name"]]
    assert len(rows) == 16 and len(grads) == 16                  # by type, and heads up to 64, 96, 128, 256; one group of waves, or two
    assert not any(k[".private_segment_fixed_size"] for k in rows)
    for k in grads:
        assert k[".private_segment_fixed_size"] <= (256 if "Li256E" in k[".name"] else 32), k[".name"]
    for name in ("rotate_axes_kernel", "append_kernel"):
        found = [k for k in kernels if name in k[".name"]]
        assert found and not any(k[".private_segment_fixed_size"] for k in found)
