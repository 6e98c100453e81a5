"""What the dense products' Python entry points refuse before anything is launched or allocated (no GPU needed)."""
import pytest
import torch

from verace_v1_b200 import linear as L

BF16 = torch.bfloat16


def meta(*shape, dt=BF16):
    return torch.empty(*shape, dtype=dt, device="meta")


@pytest.mark.parametrize("n,k", [((1 << 32) + 8, 1), (8, (1 << 32) + 8), ((1 << 24) + 1, 4), (4, (1 << 31) + 16)])
def test_sizes_beyond_the_entry_points_integers(n, k):
    """2^32 + 8 rows of weights are not 8."""
    x, w = meta(1, k), meta(n, k)
    with pytest.raises(ValueError, match="at most"):
        L._checked("fused_linear", x, w, 0, 2, None, L._ACTIVATIONS, None, BF16)
    with pytest.raises(ValueError, match="at most"):
        L._checked("gated_linear", x, w, 0, 3, "situ", L._GATES, None, BF16)


@pytest.mark.parametrize("cols", [(1 << 32) + 64, (1 << 31) + 8, (1 << 24) + 8])
def test_rows_in_8_bits_beyond_the_entry_points_integers(cols):
    with pytest.raises(ValueError, match="32768"):
        L._to_fp8("quantize_fp8", meta(1, cols), None, None, None, False)
