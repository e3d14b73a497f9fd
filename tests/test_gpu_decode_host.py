"""The native host path of rotation, cache and attention: what it binds to, and the interpreter's lock."""
import ctypes
import importlib.util
import shutil
import subprocess
import threading
import time

import pytest
import torch

from bitween_amd import PagedCache
from bitween_amd.kernels import hip_loader as hip
from test_gpu_host_path import SLOW_LIBRARY, _bind

pytestmark = pytest.mark.gpu

STEP = r"""
SLOW(bw_rotate_heads) SLOW(bw_rotate_heads_grad) SLOW(bw_cache_write) SLOW(bw_cache_read) SLOW(bw_cache_attention)
size_t bw_rotate_heads_grad_workspace_bytes() { return 0; }
size_t bw_cache_attention_workspace_bytes() { return 0; }
"""


def _copy(path, source):
    """A second copy of the native module, bound to the entry points of a C source."""
    (path / "slow.c").write_text(source)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(path / "slow.so"), str(path / "slow.c")], check=True)
    slow = ctypes.CDLL(str(path / "slow.so"))
    shutil.copy(hip._HOST_PATH, path / "_bw_host.so")
    spec = importlib.util.spec_from_file_location("slow_copy._bw_host", path / "_bw_host.so")
    host = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(host)
    _bind(host, {n: ctypes.cast(getattr(slow, n), ctypes.c_void_p).value for n in hip.ENTRY_POINTS if hasattr(slow, n)})
    return host


def _calls(host):
    cache = PagedCache(4, 1, 64, 16)
    c = (cache.keys, cache.values, None, None, 16, 0)
    q, k = torch.zeros(2, 4, 64, device="cuda").half(), torch.zeros(2, 1, 64, device="cuda").half()
    cos, slots = torch.ones(8, 32, device="cuda"), torch.tensor([1, 2], device="cuda")
    table, lengths = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    return {"rotate_heads": lambda: host.rotate_heads(q, k, cos, cos, slots, None, None, 1e-6),
            "recorded rotate_heads": lambda: host.rotate_heads(q.clone().requires_grad_(True), k, cos, cos, slots, None, None, 1e-6),
            "cache_write": lambda: host.cache_write(k, k, slots, *c), "cache_read": lambda: host.cache_read(slots, *c, hip.BW_F16),
            "cache_attention": lambda: host.cache_attention(q, table, lengths, *c, 0.125)}


def test_other_threads_run_while_a_call_is_under_way(tmp_path):
    host = _copy(tmp_path, SLOW_LIBRARY + STEP)
    ticks, stop = [0], threading.Event()

    def count():
        while not stop.is_set():
            time.sleep(0.001)
            ticks[0] += 1

    thread = threading.Thread(target=count)
    thread.start()
    try:
        for name, call in _calls(host).items():
            call()                                              # (allocator warm: the second call only sleeps)
            before, start = ticks[0], time.perf_counter()
            assert call() is not None, name
            seconds = time.perf_counter() - start
            assert seconds > 0.25 and ticks[0] - before > 20, (name, seconds, ticks[0] - before)
    finally:
        stop.set()
        thread.join()


def test_a_library_without_the_step_gives_none(tmp_path):
    for name, call in _calls(_copy(tmp_path, SLOW_LIBRARY)).items():
        assert call() is None, name
