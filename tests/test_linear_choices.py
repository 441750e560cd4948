"""Tiles and slices of the unquantized products, by the workspace that their slices take: host code only, no GPU.  Times in us
of 16-bit products, the choice that stands here and those next to it."""
import pytest

from zeromoe_amd._lib import ZmLinearDesc, lib

BF16 = 30


@pytest.mark.parametrize("S,I,O,slices", [
    (512, 4096, 4096, 4),    # 256 x 128 in four slices or 128 x 128 in four 31; 128 x 128 in two 34, whole 46
    (130, 4096, 4096, 8),    # 256 x 128 in eight 19; 128 x 128 in four 20, 256 x 128 in four 22
    (4096, 4096, 4096, 1),   # 256 x 256 141
    (8192, 1024, 8192, 1),   # 128 x 128 181; 256 x 256 304
    (2048, 4096, 1536, 2),   # 128 x 128 in two 41, whole 48
])
def test_slices_of_16_bit_products(S, I, O, slices):
    d = ZmLinearDesc(BF16, BF16, BF16, 0, S, I, O, I, I, O, O, O)
    assert lib().zm_linear_workspace_size(d) == (slices * S * O * 4 if slices > 1 else 0)
