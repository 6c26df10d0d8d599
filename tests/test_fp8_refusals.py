"""Calls of the 8-bit floating point operators that are refused, on the CPU:
scales that overlap."""
import pytest
import torch

import shady_thinker_amd as sta
from fp8_util import F8


@pytest.mark.parametrize("m,blocks,scale", [
    (3, 2, lambda: torch.ones(1, 3).expand(2, 3)),  # (a token's scale for all of its blocks)
    (1, 2, lambda: torch.ones(1, 1).expand(2, 1)),
    (3, 3, lambda: torch.ones(7).as_strided((3, 3), (2, 1)))])
def test_scales_that_overlap(m, blocks, scale):
    """A block's scales begin where the one before's end, or later: the calls
    read and write [blocks, M] of them from the first one on."""
    with pytest.raises(ValueError, match="scale"):
        sta.Fp8Rows.of(torch.zeros(m, 128 * blocks).to(F8), scale())


def test_scales_side_by_side():
    wide = torch.ones(2, 9)
    assert sta.Fp8Rows.of(torch.zeros(3, 256).to(F8), wide[:, 4:7]).stride == 9
    assert sta.Fp8Rows.of(torch.zeros(1, 256).to(F8), torch.ones(2, 1)).stride == 1
    assert sta.Fp8Rows.of(torch.zeros(3, 128).to(F8), torch.ones(3).as_strided((1, 3), (0, 1))).stride == 3  # (one block: no next one)
