"""Kernels that become resident before the one ahead of them ends: what that one writes last, and nothing runs in between,
is read as it wrote it.  Each chain is held to the same chain with a wait on the host after every call."""
import pytest
import torch
import torch.nn.functional as F

import verace_v1_b200 as V

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dt=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dt)


def unit(g, *shape, dt):
    return F.normalize(randn(g, *shape), dim=-1).to(dt)


def both(chain):
    """What the chain gives with a wait after every call, and without (three times)."""
    want = chain(torch.cuda.synchronize)
    torch.cuda.synchronize()
    for _ in range(3):
        got = chain(lambda: None)
        torch.cuda.synchronize()
        assert len(got) == len(want)
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("b", [1, 3, 64])
def test_sssd_steps_behind_one_another(b, dt):
    """Steps on one state, their inputs all there beforehand."""
    g = gen(b)
    steps, h, d = 12, 8, 128
    q, k, v = (unit(g, steps, b, h, d, dt=dt) for _ in range(3))
    dl = 0.1 * torch.rand(steps, b, h, device="cuda", generator=g)
    start = torch.eye(d, device="cuda").expand(b, h, d, d).contiguous()

    def chain(wait):
        psi, out = start.clone(), []
        wait()
        for t in range(steps):
            out.append(V.launch_decode_step((q[t], k[t], v[t], dl[t], psi), None)[0])
            wait()
        return out + [psi]
    both(chain)


@pytest.mark.parametrize("rows", [128, 8 * 128])
def test_sssd_state_from_a_product(rows):
    """A first state that a product writes, straight before the step."""
    g = gen(7)
    b, h = rows // 128, 1
    x, w = randn(g, rows, 2048, dt=BF16), randn(g, 128, 2048, dt=BF16)
    q, k, v = (unit(g, b, h, 128, dt=BF16) for _ in range(3))
    dl = 0.1 * torch.rand(b, h, device="cuda", generator=g)

    def chain(wait):
        out = []
        for i in range(4):
            psi = V.fused_linear(x, w, out_dtype=F32).view(b, h, 128, 128)
            wait()
            out += [V.launch_decode_step((q, k, v, dl, psi), None)[0], psi]
            wait()
        return out
    both(chain)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("n", [64, 128, 1024, 2048])
@pytest.mark.parametrize("maker", ["linear", "gated", "norm"])
def test_norm_weight_from_the_call_before(n, dt, maker):
    """An adaptive norm: its weight is what the call straight before it writes."""
    g = gen(n)
    k = 4096
    c, w, u = randn(g, 4, 1, k, dt=dt), randn(g, n, k, dt=dt) / 64, randn(g, n, k, dt=dt) / 64
    x = randn(g, 300, n, dt=dt)
    plain = torch.nn.RMSNorm(n, device="cuda", dtype=dt).requires_grad_(False)
    h, y = randn(g, 4, 1, n, dt=dt), randn(g, 4, 1, n, dt=dt)

    def chain(wait):
        out, sums = [], torch.zeros(4, 1, n, device="cuda", dtype=dt)
        norm = torch.nn.RMSNorm(n, device="cuda", dtype=dt).requires_grad_(False)
        wait()
        for i in range(4):
            if maker == "linear":
                made = V.fused_linear(c[i], w)
            elif maker == "gated":
                made = V.gated_linear(c[i], w, u)
            else:
                V.add_rmsnorm_fp8(h[i], y[i], plain, out=sums[i])
                made = sums[i]
            norm.weight = torch.nn.Parameter(made[0], requires_grad=False)
            wait()
            out.append(V.rmsnorm(x, norm))
            wait()
        return out
    both(chain)


@pytest.mark.parametrize("b,D,P", [(1, 128, 4), (4, 256, 8)])
@pytest.mark.parametrize("projected", [False, True])
def test_hologram_planes_from_the_call_before(b, D, P, projected):
    """The deferred hologram step straight behind what writes its planes: a product, and a flush."""
    g = gen(b + D)
    x, w = randn(g, b * D, 1024, dt=BF16), randn(g, D, 1024, dt=BF16) / 32
    q, k, v = (unit(g, b, D, dt=BF16) for _ in range(3))
    gamma = 0.1 * torch.rand(b, device="cuda", generator=g)
    rows = randn(g, b, 3 * D + 8, dt=BF16)
    empty = V.pending_storage(b, D, P)
    hi = torch.zeros(b, D, D, device="cuda")

    def chain(wait):
        pending, im, out = empty.clone(), hi.clone(), []
        wait()

        def step(re):
            if projected:
                out.append(V.launch_decode_cham_lazy_projected(rows, re, im, pending, P))
            else:
                out.append(V.launch_decode_cham_lazy(q, k, v, gamma, re, im, pending, P))
            wait()
        for i in range(3):
            re = V.fused_linear(x, w, out_dtype=F32).view(b, D, D)
            wait()
            step(re)
            step(re)
            V.decode.flush_pending(re, im, pending, P)
            wait()
            step(re)
            V.decode.flush_pending(re, im, pending, P)
            wait()
            out.append(re)
        return out + [im, pending]
    both(chain)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(300, 9000, 100), (200, 4096, 64)])
def test_partial_sums_in_chains(m, k, n, dt):
    """Sums split over K and the bias gradient's chunks, whose joins are resident while the parts are written, in workspaces
    that the calls hand on to each other."""
    g = gen(m)
    w, u, b = randn(g, n, k, dt=dt) / 64, randn(g, n, k, dt=dt) / 64, randn(g, n, dt=dt)
    x = [randn(g, m, k, dt=dt) for _ in range(4)]
    d = [randn(g, m, n, dt=dt) for _ in range(4)]

    def chain(wait):
        out = []
        for i in range(4):
            out += [V.fused_linear(x[i], w, b, activation="silu", residual=d[i]), V.gated_linear(x[i], w, u)]
            wait()
            leaves = [t.detach().requires_grad_() for t in (x[i], w, b)]
            y = V.fused_linear(*leaves, activation="gelu")
            wait()
            out += torch.autograd.grad(y, leaves, d[i])
            wait()
        return out
    both(chain)
