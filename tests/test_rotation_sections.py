"""What rotation refuses of its sections, as numbers of any size."""
import pytest
import torch

import bitween_amd as bw
from bitween_amd.kernels import hip_loader

SECTIONS = [(2 ** 70,), (16, 2 ** 63), (-(2 ** 64), 48), (2 ** 31, 16)]


def _rotate(sections, device):
    x, table = torch.zeros(4, 2, 64, dtype=torch.float16, device=device), torch.zeros(10, 32, device=device)
    bw.rotate_heads(x, x, table, table, torch.zeros(len(sections), 4, dtype=torch.int64, device=device), sections=sections)


@pytest.mark.parametrize("sections", SECTIONS)
def test_no_number_stops_the_checks(sections):
    with pytest.raises(hip_loader.BitweenHipError):              # (of CPU tensors, as with sections that fit)
        _rotate(sections, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("sections", SECTIONS)
def test_numbers_of_any_size_are_refused_alike(sections):
    with pytest.raises(ValueError, match="sections must be"):
        _rotate(sections, "cuda")
