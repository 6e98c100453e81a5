"""The dense products and the 8-bit norm in the places a program calls them from: threads, orders of calls, tensors
that other calls write."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import verace_v1_b200 as V
from linear_util import assert_within, linear64

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HERE = os.path.dirname(os.path.abspath(__file__))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def test_first_call_of_a_thread():
    """A thread whose first call of CUDA is a product (its memory comes out of the cache)."""
    g = gen(1)
    x, w, big = randn(g, 64, 256, dt=BF16), randn(g, 512, 256, dt=BF16), randn(g, 300, 256, dt=BF16)
    q4, s4, _ = V.quantize_int4(w)
    calls = [lambda: V.fused_linear(x, w), lambda: V.fused_linear(big, w), lambda: V.gated_linear(x, w, w),
             lambda: V.int4_linear(x[:8], q4, s4)]
    want = [c() for c in calls]
    for i in range(len(calls)):
        got = []

        def work():
            try:
                got.append(calls[i]())
            except Exception as e:      # (a thread's own errors reach nobody)
                got.append(e)
        calls[i]()
        torch.cuda.synchronize()
        t = threading.Thread(target=work)
        t.start()
        t.join()
        assert isinstance(got[0], torch.Tensor), got[0]
        assert torch.equal(got[0], want[i])


FIRST = """
import conftest, torch
import verace_v1_b200 as V
g = torch.Generator(device="cuda").manual_seed(2)
x, w, d = (torch.randn(*s, device="cuda", generator=g).bfloat16() for s in ((300, 128), (256, 128), (300, 256)))
torch.cuda.synchronize()
x.requires_grad_(%s), w.requires_grad_()
y = V.fused_linear(x, w)
spare = [torch.empty(1 << 22, device="cuda") for _ in range(4)]     # (what the backward asks for is in the cache)
del spare
y.backward(d)
want = d.double().t() @ x.double()
assert ((w.grad.double() - want).norm() / want.norm()) < 4e-3
print("done")
"""


@pytest.mark.parametrize("wants", [False, True])
def test_first_backward_of_a_process(wants):
    """Autograd's own thread, whose first call is a product of operands as they lie (no bias, no activation)."""
    r = subprocess.run([sys.executable, "-c", FIRST % wants], cwd=HERE, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr


def in_place_calls(x, norm):
    """(name, call) of what writes x through its pointer."""
    y = torch.ones_like(x)
    yield "add_rmsnorm_fp8", lambda: V.add_rmsnorm_fp8(x, y, norm)
    yield "add_rmsnorm_fp8 out", lambda: V.add_rmsnorm_fp8(y, y, norm, out=x)
    yield "add_rmsnorm", lambda: V.add_rmsnorm(x, y, out_norm=norm)
    rows, ids = x.view(-1, x.shape[-1]), torch.zeros(x.numel() // x.shape[-1], 1, dtype=torch.int64, device="cuda")
    yield "process_logits", lambda: V.process_logits(rows, ids, presence_penalty=0.5, out=rows)


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64)])
def test_writing_what_a_backward_has_saved_is_refused(which, shape):
    """As behind torch's own in-place operations: an input that trainable weights have read may not change before the
    backward pass has."""
    g = gen(3)
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=BF16).requires_grad_(False)
    for gated in (False, True):
        x, w, u = randn(g, *shape, dt=BF16), randn(g, 96, 64, dt=BF16).requires_grad_(), randn(g, 96, 64, dt=BF16)
        y = V.gated_linear(x, w, u) if gated else V.fused_linear(x, w)
        name, call = list(in_place_calls(x, norm))[which]
        call()
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.sum().backward()
        y = V.gated_linear(x, w, u) if gated else V.fused_linear(x, w)      # (and one without a write between is not)
        y.sum().backward()
        assert w.grad.isfinite().all()


def test_states_of_a_decode_step_count_their_versions():
    g = gen(4)
    q, k, v = (randn(g, 2, 1, 128, dt=BF16) for _ in range(3))
    psi, gate = torch.eye(128, device="cuda").expand(2, 1, 128, 128).contiguous(), torch.rand(2, 1, device="cuda", generator=g)
    re, im, pending = psi.view(2, 128, 128).clone(), torch.zeros(2, 128, 128, device="cuda"), V.pending_storage(2, 128, 4)
    was = [t._version for t in (psi, re, im, pending)]
    V.launch_decode_step((q, k, v, gate, psi), (q.view(2, 128), k.view(2, 128), v.view(2, 128), gate.view(2), re, im))
    assert psi._version > was[0] and re._version > was[1] and im._version > was[2]
    was = [t._version for t in (re, im, pending)]
    V.launch_decode_cham_lazy(q.view(2, 128), k.view(2, 128), v.view(2, 128), gate.view(2), re, im, pending, 4)
    assert all(t._version > v for t, v in zip((re, im, pending), was))
    was = [t._version for t in (re, im, pending)]
    V.flush_pending(re, im, pending, 4)
    assert all(t._version > v for t, v in zip((re, im, pending), was))
    with torch.inference_mode():        # (tensors without a version are written all the same)
        h = torch.ones(2, 64, device="cuda", dtype=BF16)
        V.add_rmsnorm_fp8(h, h, torch.nn.RMSNorm(64, device="cuda", dtype=BF16))
        assert (h == 2).all()
    V.add_rmsnorm_fp8(h, h, torch.nn.RMSNorm(64, device="cuda", dtype=BF16).requires_grad_(False))
    assert (h == 4).all()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("m", [20, 300])
def test_relu_selects_its_gradient(dt, m):
    """0 at a unit that is off, whatever the gradient is there; the gradient itself where the sum is NaN."""
    g = gen(m)
    x, w, u, d = randn(g, m, 64, dt=dt), randn(g, 96, 64, dt=dt), randn(g, 96, 64, dt=dt), randn(g, m, 96, dt=dt)
    z = x.double() @ w.double().t()
    sure = z.abs() > 0.01
    d = torch.where(sure, d, torch.zeros_like(d))
    off = (z < 0) & sure
    clean = torch.autograd.grad(V.fused_linear(*(t := [x.clone().requires_grad_(), w.clone().requires_grad_()]), activation="relu"), t, d)
    bad = d.clone()
    bad[off & (torch.rand(m, 96, device="cuda", generator=g) < 0.2)] = float("inf")
    bad[off & (torch.rand(m, 96, device="cuda", generator=g) < 0.2)] = float("nan")
    got = torch.autograd.grad(V.fused_linear(*t, activation="relu"), t, bad)
    assert all(torch.equal(a, b) for a, b in zip(got, clean)) and all(a.isfinite().all() for a in got)
    # the gate's gradient likewise (the up projection's is d relu(g): NaN of an infinite d, as torch's product is)
    t = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    got, = torch.autograd.grad(V.gated_linear(t[0], t[1], u, activation="relu"), t[1], bad)
    want, = torch.autograd.grad(V.gated_linear(t[0], t[1], u, activation="relu"), t[1], d)
    assert torch.equal(got, want) and got.isfinite().all()
    # a row of NaN sums: the weights as they are in x's gradient
    x2 = x.clone()
    x2[3, 5] = float("nan")
    t = [x2.requires_grad_(), w]
    got, = torch.autograd.grad(V.fused_linear(*t, activation="relu"), t[0], d)
    plain, = torch.autograd.grad(V.fused_linear(*t), t[0], d)
    assert torch.equal(got[3], plain[3]) and torch.equal(got[[i for i in range(m) if i != 3]], clean[0][[i for i in range(m) if i != 3]])


def test_derivatives_that_nobody_would_get_are_refused():
    """Scales that require a gradient, and forward-mode tangents of any operand."""
    import torch.autograd.forward_ad as ad
    g = gen(6)
    x, w, b, r = randn(g, 5, 64, dt=BF16), randn(g, 32, 64, dt=BF16), randn(g, 32, dt=BF16), randn(g, 5, 32, dt=BF16)
    (q, s), (wq, ws) = V.quantize_fp8(x), V.quantize_fp8(w)
    for i in range(2):
        sc = [s.clone(), ws.clone()]
        sc[i].requires_grad_()
        with pytest.raises(RuntimeError, match="no_grad"):
            V.fused_linear(q, wq, x_scale=sc[0], w_scale=sc[1])
        with torch.no_grad():
            V.fused_linear(q, wq, x_scale=sc[0], w_scale=sc[1])
    for i in range(3):
        sc = [s.clone(), ws.clone(), ws.clone()]
        sc[i].requires_grad_()
        with pytest.raises(RuntimeError, match="no_grad"):
            V.gated_linear(q, wq, wq, x_scale=sc[0], gate_scale=sc[1], up_scale=sc[2])
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=BF16).requires_grad_(False)
    with ad.dual_level():
        def dual(t):
            return ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: V.fused_linear(dual(x), w), lambda: V.fused_linear(x, dual(w)), lambda: V.fused_linear(x, w, dual(b)),
                     lambda: V.fused_linear(x, w, residual=dual(r)), lambda: V.gated_linear(dual(x), w, w),
                     lambda: V.gated_linear(x, w, dual(w)), lambda: V.quantize_fp8(dual(x)), lambda: V.rmsnorm_fp8(dual(x), norm),
                     lambda: V.fused_linear(q, wq, x_scale=dual(s), w_scale=ws),
                     lambda: V.add_rmsnorm_fp8(x.clone(), dual(x), norm)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        V.fused_linear(x, w)            # (no operand with a tangent)


def test_a_quantised_model_in_another_type():
    """model.half() behind quantize_model_fp8: the same 8-bit weights, fp16 in and out."""
    from test_fp8_model_gpu import make_model
    model = V.quantize_model_fp8(make_model(BF16))
    moe = model.layers[0].mcmoe
    up, down = moe.base_situ_glu.fp8_in.w_up.clone().view(torch.uint8), moe.base_w_down.scales.clone()
    model.half()
    assert torch.equal(moe.base_situ_glu.fp8_in.w_up.view(torch.uint8), up) and torch.equal(moe.base_w_down.scales, down)
    ids = torch.randint(0, 101, (2, 5), generator=torch.Generator().manual_seed(1)).cuda()
    tokens, lp = V.generate(model, ids, 3)
    assert tokens.shape == (2, 8) and lp.isfinite().all()
    with torch.no_grad():
        logits, _, _ = model(ids, return_layer_states=True)
        x = randn(gen(8), 1, 4, 128, dt=F16)
        q, s = V.quantize_fp8(x)
        f = moe.base_situ_glu.fp8_in
        assert torch.equal(f(x), V.gated_linear(q, f.w_gate, f.w_up, x_scale=s, gate_scale=f.gate_scales, up_scale=f.up_scales,
                                                out_dtype=F16))
    assert logits.dtype is F16 and logits.isfinite().all()
    model.float()
    assert V.generate(model, ids, 2)[1].isfinite().all() and model.lm_head.dtype is F32


@pytest.mark.parametrize("handed_on", [False, True])
def test_hooks_of_the_base_block_see_its_8_bit_calls(handed_on):
    from test_fp8_model_gpu import make_model
    moe = V.quantize_model_fp8(make_model(BF16)).layers[1].mcmoe
    x = randn(gen(9), 2, 3, 128, dt=BF16)
    x8 = V.quantize_fp8(x) if handed_on else None
    with torch.no_grad():
        want = moe(x, x8)
        seen = []
        handles = [moe.base_situ_glu.register_forward_pre_hook(lambda m, a: seen.append(len(a))),
                   moe.base_situ_glu.register_forward_hook(lambda m, a, out: out * 0)]
        without = moe(x, x8)
        assert seen == [2 if handed_on else 1] and not torch.equal(without, want)
        for h in handles:
            h.remove()
        assert torch.equal(moe(x, x8), want)


def test_a_model_that_cannot_go_into_8_bits_stays_as_it_is():
    from test_fp8_model_gpu import make_model
    for spoil in (lambda m: setattr(m.layers[2].mcmoe, "base_w_down", torch.nn.Linear(40000, 128, bias=False, device="cuda")),
                  lambda m: m.layers[1].mcmoe.base_w_down.cpu(), lambda m: m.lm_head.double()):
        model = make_model(BF16)
        spoil(model)
        with pytest.raises((ValueError, AssertionError)):
            V.quantize_model_fp8(model)
        for layer in model.layers:
            assert layer.mcmoe.base_situ_glu.w_gate is not None and layer.mcmoe.base_situ_glu.fp8_in is None
            assert isinstance(layer.mcmoe.base_w_down, torch.nn.Linear)
        assert isinstance(model.lm_head, torch.nn.Linear)


def test_a_sum_is_not_written_over_a_leaf():
    norm = torch.nn.RMSNorm(64, device="cuda", dtype=BF16).requires_grad_(False)
    h, y = torch.ones(3, 64, device="cuda", dtype=BF16), torch.ones(3, 64, device="cuda", dtype=BF16)
    out = torch.zeros(3, 64, device="cuda", dtype=BF16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        V.add_rmsnorm_fp8(h, y, norm, out=out)
    assert not out.any()
    with torch.no_grad():
        V.add_rmsnorm_fp8(h, y, norm, out=out)
    assert (out == 2).all()


def back_and_forth(t):
    """A saved tensor, as a hook may keep it: another tensor of the same values, dense."""
    return t.clone(memory_format=torch.contiguous_format)


def columns_first(t):
    """Dense along the other dimension."""
    return t.t().contiguous().t() if t.dim() == 2 else t.clone()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("m", [4, 130, 300])
@pytest.mark.parametrize("hooks", [(back_and_forth, back_and_forth), (columns_first, lambda t: t), "cpu"])
def test_what_was_saved_comes_back_in_another_layout(dt, m, hooks):
    """Operands inside of wider tensors, whose saved rows come back dense, or transposed, behind hooks."""
    g = gen(m)
    wide, ww, d = randn(g, m, 200, dt=dt), randn(g, 96, 300, dt=dt), randn(g, m, 96, dt=dt)

    def grads():
        x, w, u = (t.detach().requires_grad_() for t in (wide[:, 8:136], ww[:, 16:144], ww[:, 160:288]))
        y, h = V.fused_linear(x, w, activation="silu"), V.gated_linear(x, w, u)
        return torch.autograd.grad(y, (x, w), d) + torch.autograd.grad(h, (x, w, u), d)
    want = grads()
    if hooks == "cpu":
        with torch.autograd.graph.save_on_cpu():
            got = grads()
    else:
        with torch.autograd.graph.saved_tensors_hooks(*hooks):
            got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("shape", [(64,), (6, 64), (2, 3, 64), (2, 1, 3, 64), (0, 3, 64)])
def test_outputs_may_be_changed_in_place(shape):
    """As torch.nn.functional.linear's may, in any number of dimensions."""
    g = gen(11)
    x, w, r = randn(g, *shape), randn(g, 96, 64), randn(g, *shape[:-1], 96)
    for call in (lambda a, b: V.fused_linear(a, b), lambda a, b: V.gated_linear(a, b, w)):
        got = [t.clone().requires_grad_() for t in (x, w)]
        want = [t.clone().requires_grad_() for t in (x, w)]
        y = call(*got)
        assert y.shape == shape[:-1] + (96,)
        y.mul_(r)
        y += 1
        y.sum().backward()
        (call(*want) * r + 1).sum().backward()
        assert all(torch.equal(a.grad, b.grad) and a.grad.shape == b.shape for a, b in zip(got, want))


def test_another_module_in_the_sub_layers_place():
    """A layer whose feed-forward sub-layer, or its base block, a user has replaced or wrapped."""
    from test_fp8_model_gpu import make_model

    class Wrapped(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x):
            return self.inner(x)
    x = randn(gen(12), 2, 5, 128, dt=BF16)
    for eight in (False, True):
        layer = make_model(BF16).layers[1]
        if eight:
            V.quantize_model_fp8(layer)
        with torch.no_grad():
            want = layer(x)[0]
            inner = layer.mcmoe
            layer.mcmoe = Wrapped(inner)
            # (in 8 bits the sub-layer then quantises the norm's rounded rows itself)
            assert torch.equal(layer(x)[0], want) or eight and layer(x)[0].isfinite().all()
            layer.mcmoe = torch.nn.Linear(128, 128, device="cuda", dtype=BF16)
            assert layer(x)[0].isfinite().all()
            layer.mcmoe = inner
            inner.base_situ_glu = torch.nn.Linear(128, inner.base_w_down.in_features, device="cuda", dtype=BF16)
            assert layer(x)[0].isfinite().all()
