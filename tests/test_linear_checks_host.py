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


def filled(m):
    g = torch.Generator().manual_seed(1)
    for name, t in m.named_buffers():
        if t.dtype is torch.float8_e4m3fn:
            t.copy_((torch.randn(t.shape, generator=g) * 50).to(t.dtype))
        else:
            t.copy_(torch.rand(t.shape, generator=g))
    return m


@pytest.mark.parametrize("make", [lambda: L.Fp8Linear(24, 16, True), lambda: L.Fp8Linear(24, 16), lambda: L.Fp8GatedLinear(24, 16)])
@pytest.mark.parametrize("change,dtype", [(lambda m: m.half(), torch.float16), (lambda m: m.float(), torch.float32),
                                          (lambda m: m.to(torch.float16), torch.float16), (lambda m: m.bfloat16(), BF16),
                                          (lambda m: m.to("cpu"), BF16), (lambda m: m.type(torch.float16), torch.float16),
                                          (lambda m: m.to(torch.float32).to(BF16), BF16)])
def test_8_bit_modules_keep_their_weights_when_their_type_changes(make, change, dtype):
    m = filled(make())
    was = {name: t.clone() for name, t in m.named_buffers()}
    holder = torch.nn.Sequential(m)
    assert change(holder) is holder and m.dtype is dtype and list(m.state_dict()) == list(was)
    for name, t in m.named_buffers():
        if name == "bias":
            assert t.dtype is dtype
        else:
            assert t.dtype is was[name].dtype and torch.equal(t.float(), was[name].float())


def test_8_bit_modules_without_memory():
    m = L.Fp8Linear(24, 16, True, device="meta").half()
    assert m.weight.dtype is torch.float8_e4m3fn and m.scales.dtype is torch.float32 and m.bias.dtype is torch.float16
    m = m.to_empty(device="cpu")
    assert m.weight.device.type == "cpu" and m.weight.dtype is torch.float8_e4m3fn and m.scales.shape == (16,)
    m = filled(L.Fp8GatedLinear(24, 16)).to("meta")
    assert m.w_up.is_meta and m.w_up.dtype is torch.float8_e4m3fn and m.dtype is BF16
