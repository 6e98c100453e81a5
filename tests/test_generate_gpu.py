"""The generation loop: the 4-bit products, the logits' processing and the choice of a token as
they run together, on a small VeraceV1Model.

The quantised model is compared with the same model holding the dequantised weights: fp32 on
both sides, so a projection differs by its sums' rounding (4e-6 in the 2-norm, see
test_int4_gpu.py) and the logits after four layers of normalised activations by the reference
tests' rtol 1e-3 / atol 1e-4."""
import pytest
import torch

import verace_v1_b200 as V
from conftest import model_reinit

pytestmark = pytest.mark.gpu


def make_model(dtype=torch.float32):
    cfg = V.VeraceV1Config(vocab_size=100, hidden_dim=128, num_layers=4, num_heads=1, head_dim=128, spectral_dim=64,
                           chams_holographic_dim=128, mcmoe_rank=8, mcmoe_num_components=8)
    model = V.VeraceV1Model(cfg).eval()
    model_reinit(model, seed=0)
    return model.cuda().to(dtype)


def prompt(b=3, s=7):
    return torch.randint(0, 100, (b, s), generator=torch.Generator().manual_seed(1)).cuda()


def test_greedy_matches_argmax_loop():
    model, ids = make_model(), prompt()
    tokens, lp = V.generate(model, ids, 6)
    assert tokens.shape == (3, 13) and lp.shape == (3, 6) and torch.equal(tokens[:, :7], ids)
    with torch.no_grad():
        logits, _, st = model(ids, return_layer_states=True)
        for i in range(6):
            want = logits[:, -1].argmax(-1)
            assert torch.equal(tokens[:, 7 + i], want)
            ref = torch.log_softmax(logits[:, -1].double(), -1).gather(1, want[:, None])[:, 0]
            assert ((lp[:, i] - ref).abs() <= 1e-5).all()
            logits, _, st = model(want[:, None], layer_states=st, return_layer_states=True)


def test_quantised_model_matches_its_dequantised_weights():
    ids = prompt()
    a, b = make_model(), make_model()
    V.quantize_model_int4(a, group_size=64, symmetric=False)
    assert not [n for n, m in a.named_modules() if isinstance(m, torch.nn.Linear) and "router" not in n
                and "w_halting" not in n], "a projection is still dense"
    for x, y in zip(a.layers, b.layers):
        for p, q, names in ((x.sssd_attn, y.sssd_attn, ("w_q", "w_k", "w_v", "w_delta")),
                            (x.cham_memory, y.cham_memory, ("w_q", "w_k", "w_v", "w_gamma")),
                            (x.mcmoe.base_situ_glu, y.mcmoe.base_situ_glu, ("w_gate", "w_up"))):
            w, at = p.int4_in.dequantized(), 0
            for name in names:
                lin = getattr(q, name)
                lin.weight.data.copy_(w[at:at + lin.weight.shape[0]])
                at += lin.weight.shape[0]
        for p, q in ((x.sssd_attn.w_out, y.sssd_attn.w_out), (x.cham_memory.w_out, y.cham_memory.w_out),
                     (x.mcmoe.base_w_down, y.mcmoe.base_w_down), (x.mcmoe.hyper_sigma, y.mcmoe.hyper_sigma)):
            q.weight.data.copy_(p.dequantized())
    b.embed_tokens.weight = torch.nn.Parameter(a.embed_tokens.weight.detach().clone())
    b.lm_head.weight = torch.nn.Parameter(a.lm_head.dequantized())
    with torch.no_grad():
        la, _, sa = a(ids, return_layer_states=True)
        lb, _, sb = b(ids, return_layer_states=True)
        torch.testing.assert_close(la, lb, rtol=1e-3, atol=1e-4)
        la, _, _ = a(ids[:, :1], layer_states=sa, return_layer_states=True)
        lb, _, _ = b(ids[:, :1], layer_states=sb, return_layer_states=True)
        torch.testing.assert_close(la, lb, rtol=1e-3, atol=1e-4)
    ta, _ = V.generate(a, ids, 4)
    tb, _ = V.generate(b, ids, 4)
    assert torch.equal(ta, tb)
    assert V.device_status() == 0


def test_rows_that_biases_leave_nothing_end():
    model, ids = make_model(), prompt()
    everything = torch.arange(100, device="cuda").expand(3, 100).contiguous()
    values = torch.zeros(3, 100, device="cuda")
    values[1] = -float("inf")
    tokens, lp = V.generate(model, ids, 4, bias_ids=everything, bias_values=values)
    want, want_lp = V.generate(model, ids, 4)
    assert torch.equal(tokens[[0, 2]], want[[0, 2]])
    torch.testing.assert_close(lp[[0, 2]], want_lp[[0, 2]], rtol=1e-3, atol=1e-4)
    assert (tokens[1, 7:] == -1).all() and (lp[1] == 0).all()


def test_controls_and_ends_of_rows():
    model, ids = make_model(torch.bfloat16), prompt()
    V.quantize_model_int4(model, group_size=128)
    g = torch.Generator(device="cuda").manual_seed(3)
    kw = dict(temperature=0.8, top_k=20, top_p=0.9, repetition_penalty=1.3, frequency_penalty=0.1)
    a = V.generate(model, ids, 5, generator=g, **kw)
    g.manual_seed(3)
    b = V.generate(model, ids, 5, generator=g, **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and ((a[0] >= 0) & (a[0] < 100)).all()
    # a grammar: only token 10 + i at step i, and nothing for row 1 from step 2 on
    def grammar(so_far):
        i = so_far.shape[1] - 7
        words = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
        words[:, 0] = 1 << (10 + i)
        if i >= 2:
            words[1] = 0
        return words
    tokens, lp = V.generate(model, ids, 4, allowed=grammar)
    assert tokens[0, 7:].tolist() == tokens[2, 7:].tolist() == [10, 11, 12, 13]
    assert tokens[1, 7:].tolist() == [10, 11, -1, -1] and (lp[1, 2:] == 0).all()
    # a bias that makes one token certain, and it ends the rows
    tokens, _ = V.generate(model, ids, 9, eos_token_id=42, bias_ids=torch.full((3, 1), 42, device="cuda"),
                           bias_values=torch.full((3, 1), 1e4, device="cuda"))
    assert tokens.shape == (3, 8) and (tokens[:, 7] == 42).all()
    assert V.generate(model, ids, 0)[0].shape == (3, 7)
