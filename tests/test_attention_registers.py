"""Registers of the attention kernels that go to memory, from the built library's metadata."""
import re

from bitween_amd.kernels import hip_loader
from test_abi_and_host import _kernel_metadata

# (bits, groups of a head, queries of a segment up to): groups of 32, whose pairs, reaches and sums all live at once
SPILLED = {(8, 8, 4), (8, 8, 8), (8, 8, 16), (8, 7, 4), (8, 7, 8), (8, 7, 16), (8, 6, 16), (8, 4, 8), (8, 4, 16), (4, 8, 4), (4, 8, 8), (4, 8, 16), (4, 7, 8), (4, 7, 16),
           (4, 4, 16), (4, 2, 8), (4, 2, 16)}


def test_attention_kernels_spill_in_groups_of_32_only():
    """16 bits, groups of 64 and 128, and up to 4 queries over heads of up to 192 in groups of 32 keep everything in registers; the others no more than they did."""
    kernels = [k for k in _kernel_metadata(hip_loader.library_path()) if "attention_kernel" in k[".name"]]
    assert len(kernels) == 6 + 2 * 3 * (8 + 4 + 2)               # 16 bits by type and head; codes by queries and groups
    for k in kernels:
        spilled = k[".private_segment_fixed_size"] or k[".vgpr_spill_count"]
        m = re.search(r"FormatQILi(\d)ELi(\d)ELi(\d+)EELi(\d)", k[".name"])
        if m is None:
            assert not spilled, k[".name"]
            continue
        bits, groups, size, fold = map(int, m.groups())
        assert not spilled or size == 32 and (bits, groups, 16 // fold) in SPILLED, k[".name"]
        assert k[".private_segment_fixed_size"] <= 700, k[".name"]
