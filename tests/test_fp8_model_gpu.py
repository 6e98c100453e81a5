"""The 8-bit feed-forward sub-layer as the framework's own modules run it (quantize_model_fp8): the M-CMoE,
a decoder layer and the generation loop."""
import pytest
import torch

import verace_v1_b200 as V
from conftest import model_reinit
from linear_util import assert_within, dequantised, gated64, linear64

pytestmark = pytest.mark.gpu


def make_model(dtype):
    cfg = V.VeraceV1Config(vocab_size=101, hidden_dim=128, num_layers=3, num_heads=1, head_dim=128, spectral_dim=64,
                           chams_holographic_dim=128, mcmoe_rank=8, mcmoe_num_components=8)
    model = V.VeraceV1Model(cfg).eval()
    model_reinit(model, seed=0)
    return model.cuda().to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 9, 150])
def test_mcmoe_in_8_bits(dtype, tokens):
    """The module's output is the operators' on its buffers; the base block is held to the formulas."""
    m = make_model(dtype).layers[0].mcmoe
    dense = {k: getattr(m.base_situ_glu, k).weight.detach().double() for k in ("w_gate", "w_up")}
    V.quantize_model_fp8(m)
    g8 = m.base_situ_glu.fp8_in
    assert m.base_situ_glu.w_gate is None and isinstance(m.base_w_down, V.Fp8Linear)
    for name, scale in (("w_gate", g8.gate_scales), ("w_up", g8.up_scales)):   # weights within half an e4m3 step
        w = dequantised(getattr(g8, name), scale)
        assert ((w - dense[name]).abs() <= 2.0 ** -4 * dense[name].abs() + 2.0 ** -9 * scale.double()[:, None]).all()
    x = torch.randn(1, tokens, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(tokens)).to(dtype)
    with torch.no_grad():
        got = m(x)
        flat = x.view(tokens, 128)
        q, s = V.quantize_fp8(flat)
        h = g8((q, s))
        assert_within(h, gated64(dequantised(q, s), dequantised(g8.w_gate, g8.gate_scales),
                                 dequantised(g8.w_up, g8.up_scales), "situ", dtype))
        assert torch.equal(g8(flat), h)
        idx, w = V.launch_mcmoe_route(m.router(flat), 8)
        manifold = V.rmsnorm(V.launch_mcmoe_projection(flat, m.u_basis, m.v_basis, idx, w, m.hyper_sigma(flat),
                                                       sigma_is_logits=True), m.norm)
        qh, sh = V.quantize_fp8(h)
        down = m.base_w_down
        want = V.fused_linear(qh, down.weight, residual=manifold, x_scale=sh, w_scale=down.scales, out_dtype=dtype)
        assert_within(want, linear64(dequantised(qh, sh), dequantised(down.weight, down.scales), None, None, manifold, dtype))
        assert torch.equal(got.view(tokens, 128), want)
        assert torch.equal(m(x, (q, s)), got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_hands_its_norm_on_in_8_bits(dtype):
    """The layer's fused step gives the sub-layer the norm in its own type and the same rows in 8 bits."""
    layer = make_model(dtype).layers[1]
    V.quantize_model_fp8(layer)
    seen = []
    inner = layer.mcmoe.forward
    layer.mcmoe.forward = lambda n, x8=None: (seen.append((n.clone(), x8)), inner(n, x8))[1]
    x = torch.randn(2, 5, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    with torch.no_grad():
        out = layer(x)[0]
    (n, (q, s)), = seen
    assert out.shape == x.shape and out.isfinite().all() and q.shape == n.shape and s.shape == n.shape[:-1]
    v = n.double() / s.double()[..., None]
    # half an e4m3 step of the value before its rounding to the type, which is within half a step of the type of n
    e = torch.finfo(dtype).eps
    assert ((q.double() - v).abs() <= torch.clamp(v.abs() * (2.0 ** -4 + e), min=2.0 ** -10) + e * v.abs()).all()


def test_generation_in_8_bits():
    model = make_model(torch.bfloat16)
    V.quantize_model_fp8(model)
    ids = torch.randint(0, 101, (3, 6), generator=torch.Generator().manual_seed(1)).cuda()
    tokens, lp = V.generate(model, ids, 5)
    assert tokens.shape == (3, 11) and lp.isfinite().all() and ((tokens >= 0) & (tokens < 101)).all()
    with torch.no_grad():
        logits, _, _ = model(ids, return_layer_states=True)
    assert logits.dtype is torch.bfloat16 and torch.equal(tokens[:, 6], logits[:, -1].float().argmax(-1))
    V.quantize_model_int4(model)         # the rest in 4 bits beside it
    assert model.layers[0].mcmoe.base_situ_glu.int4_in is None and isinstance(model.lm_head, V.Fp8Linear)
    tokens, lp = V.generate(model, ids, 2)
    assert tokens.shape == (3, 8) and lp.isfinite().all()
    assert V.device_status() == 0


def test_modules_keep_their_state():
    lin = torch.nn.Linear(40, 24, device="cuda", dtype=torch.float16)
    a = V.Fp8Linear.from_linear(lin)
    b = V.Fp8Linear(40, 24, True, torch.float16, device="cuda")
    b.load_state_dict(a.state_dict())
    x = torch.randn(3, 40, device="cuda", dtype=torch.float16)
    with torch.no_grad():
        assert torch.equal(a(x), b(x)) and torch.equal(a(V.quantize_fp8(x)), a(x))
        r = torch.randn(3, 24, device="cuda", dtype=torch.float16)
        q, s = V.quantize_fp8(x)
        assert_within(a(x, residual=r, activation="silu"),
                      linear64(dequantised(q, s), dequantised(a.weight, a.scales), a.bias, "silu", r, torch.float16))
    g = V.Fp8GatedLinear.from_weights(lin.weight, lin.weight, "silu")
    h = V.Fp8GatedLinear(40, 24, "silu", dtype=torch.float16, device="cuda")
    h.load_state_dict(g.state_dict())
    with torch.no_grad():
        assert torch.equal(g(x), h(x))
