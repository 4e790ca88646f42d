"""The trainers' feed-forward operators on the CPU: argument checks, the plain forms against their formulas and against
differences, the generator against published vectors, and the paths that call them (LoRA dropout through checkpointing,
the SFT command, the opt-in feed-forward)."""
import json

import pytest
import torch

from arc_forge_2026_b200.config import preset
from arc_forge_2026_b200.train import fused, kernels, lora, sft
from arc_forge_2026_b200.train.ffn import gated_ffn, gated_ffn_reference

BF = torch.bfloat16


def test_gated_ffn_refuses_what_does_not_fit():
    x, w13, w2 = torch.zeros(3, 16), torch.zeros(16, 16), torch.zeros(24, 8)
    assert gated_ffn(x, w13, w2).shape == (3, 24)
    assert gated_ffn(x.view(1, 3, 16), w13, w2, act="gelu", residual=torch.ones(1, 3, 24)).eq(1).all()
    for kw in (dict(act="relu"), dict(w13=torch.zeros(18, 16)), dict(w13=torch.zeros(16, 8)),
               dict(w2=torch.zeros(24, 16)), dict(w2=torch.zeros(8)), dict(w2=torch.zeros(24, 8, dtype=BF)),
               dict(w13=torch.zeros(16, 16, dtype=BF)), dict(residual=torch.zeros(3, 16)),
               dict(residual=torch.zeros(1, 24)), dict(residual=torch.zeros(3, 24, dtype=BF)),
               dict(x=torch.zeros(3, 0), w13=torch.zeros(16, 0)), dict(w13=torch.zeros(0, 16), w2=torch.zeros(24, 0)),
               dict(w13=torch.zeros(16, 16, device="meta"))):
        with pytest.raises(ValueError):
            gated_ffn(**{**dict(x=x, w13=w13, w2=w2), **kw})


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu"])
def test_gated_ffn_plain_form(act):
    g = torch.Generator().manual_seed(0)
    x, w13, w2, r = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
                     for s in ((5, 6), (8, 6), (3, 4), (5, 3)))
    gate, up = x @ w13[:4].T, x @ w13[4:].T
    a = {"silu": gate * torch.sigmoid(gate), "gelu": 0.5 * gate * (1 + torch.erf(gate / 2 ** 0.5)),
         "gelu_tanh": 0.5 * gate * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (gate + 0.044715 * gate ** 3)))}[act]
    assert torch.allclose(gated_ffn(x, w13, w2, act, r), (a * up) @ w2.T + r, rtol=1e-12)
    assert torch.autograd.gradcheck(lambda *t: gated_ffn_reference(t[0], t[1], t[2], act, t[3]), (x, w13, w2, r))


def test_layer_norm_plain_form_and_refusals():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 5, 12, generator=g, dtype=torch.float64, requires_grad=True)
    w, b = (torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    assert torch.allclose(fused.layer_norm(x, w, b, 1e-6),
                          torch.nn.functional.layer_norm(x, (12,), w, b, 1e-6), rtol=1e-10)
    assert torch.autograd.gradcheck(lambda *t: fused.layer_norm(*t, 1e-6), (x, w, b))
    y = fused.layer_norm(x.detach().to(BF), w.detach().float(), None, 1e-6)
    assert y.dtype == BF
    for args in ((x, w[:11]), (x, w, b[:11]), (x, w[None]), (x, w, b.float()), (x, w.to("meta")),
                 (x, w, b.to("meta"))):
        with pytest.raises(ValueError):
            fused.layer_norm(*args)


# Philox4x32-10 known answers (counter words, key words, output words) of the generator's published test vectors
KAT = [((0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8))]


def test_generator_known_answer():
    for (c0, c1), (k0, k1), out in KAT:
        seed, ctr = k0 | k1 << 32, c0 | c1 << 32
        words = [v for w in out for v in (w & 0xFFFF, w >> 16)]
        # the threshold at which each element changes is its 16 bits
        for i, v in enumerate(words):
            for t, kept in ((v, False), (v + 1, True)):
                p = 1 - t / 65536
                assert fused.dropout_threshold(p) == t
                assert bool(fused.dropout_keep_reference(8, p, seed, ctr)[i]) == kept


def test_dropout_plain_form():
    x = torch.randn(1000, 33, generator=torch.Generator().manual_seed(2))
    y = fused.dropout(x, 0.25, 7)
    kept = y != 0
    assert abs(kept.double().mean().item() - 0.75) < 5 * (0.25 * 0.75 / x.numel()) ** 0.5  # five standard deviations
    assert torch.equal(y[kept], (x * (65536 / 49152))[kept])
    # the counter counts blocks of eight elements: an offset is a shift of the mask
    flat = fused.dropout_keep_reference(8000, 0.25, 7)
    assert torch.equal(fused.dropout_keep_reference(7992, 0.25, 7, 1), flat[8:])
    assert not torch.equal(fused.dropout_keep_reference(8000, 0.25, 8), flat)
    # counters pass 2^32 and seeds are taken modulo 2^64
    a = fused.dropout_keep_reference(64, 0.5, 3, 2 ** 32 - 4)
    assert torch.equal(a[32:], fused.dropout_keep_reference(32, 0.5, 3, 2 ** 32))
    assert torch.equal(fused.dropout(x, 0.5, -1), fused.dropout(x, 0.5, 2 ** 64 - 1))
    # gradient: the mask times the scale; the residual's is the incoming one
    lx, lr = x.clone().requires_grad_(True), torch.ones_like(x).requires_grad_(True)
    out = fused.dropout(lx, 0.25, 7, residual=lr)
    assert torch.equal(out.detach(), y + 1)
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(3))
    dx, dr = torch.autograd.grad(out, [lx, lr], dy)
    assert torch.equal(dx, torch.where(kept, dy * (65536 / 49152), 0.0)) and torch.equal(dr, dy)
    # everything, nothing, infinities in dropped places
    assert torch.equal(fused.dropout(x, 0.0, 7), x) and not fused.dropout(x, 1.0, 7).any()
    assert torch.equal(fused.dropout(x.masked_fill(~kept, float("inf")), 0.25, 7), y)
    assert torch.equal(fused.dropout(x, 0.25, torch.tensor([5, 1]), -1), fused.dropout(x, 0.25, 5))
    for kw in (dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(residual=x[:1]), dict(residual=x.to(BF)),
               dict(seed=torch.tensor([1.0, 2.0])), dict(seed=torch.tensor([1])), dict(x=torch.ones(3).int())):
        with pytest.raises(ValueError):
            fused.dropout(**{**dict(x=x, p=0.1, seed=1), **kw})


def _student(dropout, checkpoint_layers=True):
    from arc_forge_2026_b200.train.student import random_student
    st = random_student(preset("tiny_cpu"), "cpu", seed=0, checkpoint_layers=checkpoint_layers)
    lora.attach_lora(st, 8, 16.0, seed=3, dropout=dropout)
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for layer in st.layers:
            for ad in layer.lora.values():
                ad.B.copy_(torch.randn(ad.B.shape, generator=g) * 0.05)
    return st


def test_lora_dropout_masks_are_recomputed_not_redrawn():
    ids = torch.randint(0, 200, (1, 64), generator=torch.Generator().manual_seed(4))

    def grads(st, step):
        lora.set_dropout_step(st, step)
        ps = [p for p in st.parameters() if p.requires_grad]
        return torch.autograd.grad(st.hidden(ids).float().square().sum(), ps)
    a, b = _student(0.2), _student(0.2, checkpoint_layers=False)
    for u, v in zip(grads(a, 7), grads(b, 7)):  # the checkpointed layers drop the same elements again
        assert torch.equal(u, v)
    assert any(not torch.equal(u, v) for u, v in zip(grads(a, 7), grads(a, 8)))
    seeds = [ad.dropout_seed for layer in a.layers for ad in layer.lora.values()]
    assert len(set(seeds)) == len(seeds)
    a.eval()
    none = _student(0.0)
    assert torch.equal(a.hidden(ids), none.hidden(ids))
    with pytest.raises(ValueError):
        lora.set_dropout_step(a, -1)
    with pytest.raises(ValueError):
        lora.attach_lora(_student(0.0), dropout=1.0)


def test_sft_with_lora_dropout_resumes_on_the_same_masks(tmp_path, capsys):
    d = tmp_path / "d.jsonl"
    g = torch.Generator().manual_seed(6)
    d.write_text("".join(json.dumps({"ids": torch.randint(1, 200, (50,), generator=g).tolist()}) + "\n"
                         for _ in range(4)))

    def run(out, steps, *extra):
        sft.main(["--data", str(d), "--preset", "tiny_cpu", "--max-len", "128", "--bins-per-step", "2", "--lora-r", "8",
                  "--out", str(tmp_path / out), "--steps", str(steps), "--lora-dropout", "0.3", *extra])
        return [json.loads(x)["loss"] for x in capsys.readouterr().out.splitlines() if x.startswith('{"step"')]
    whole = run("a", 4)
    assert run("b", 2) + run("b", 4, "--resume") == whole


def test_opt_in_feed_forward_leaves_cpu_runs_alone():
    old = {n for n in kernels.NAMES if kernels.enabled(n)}
    ids = torch.randint(0, 200, (1, 64), generator=torch.Generator().manual_seed(7))
    st = _student(0.0)
    y = st.hidden(ids)
    try:
        assert "gated_ffn" not in kernels.enable("all") and {"layer_norm", "dropout"} <= kernels.enable("all")
        kernels.enable(sorted(old | {"gated_ffn"}))
        assert torch.equal(st.hidden(ids), y)
    finally:
        kernels.enable(sorted(old))


def test_tensors_without_memory_never_reach_the_kernels():
    """A fake tensor says that it is on the GPU and has no memory; function-transform wrappers and lazily negated views
    have memory that is not their value. The bindings leave them to the plain forms before they look at any pointer, and
    so they do inside transforms, dispatch modes and traces."""
    pytest.importorskip("arc_forge_2026_b200._C")
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    from arc_forge_2026_b200.ops import C
    ext = C()
    for dt in (torch.float32, BF):
        with FakeTensorMode():
            x, w = torch.empty(6, 40, dtype=dt, device="cuda"), torch.empty(40, device="cuda")
            w13, w2 = torch.empty(32, 40, dtype=dt, device="cuda"), torch.empty(24, 16, dtype=dt, device="cuda")
            for t in (x, x.detach().requires_grad_(True)):
                assert t.is_cuda and fused.rms_norm(t, w, 1e-6).shape == fused.layer_norm(t, w).shape == (6, 40)
                assert fused.dropout(t, 0.5, 1).shape == (6, 40) and gated_ffn(t, w13, w2).shape == (6, 24)
                assert fused.rms_norm(t, w, 1e-6).requires_grad == t.requires_grad
        assert ext.train_norm(x, w, None, 1e-6, True) is None and ext.dropout(x, None, 9, 1, 1, None) is None
        assert ext.gated_ffn(x, w13, w2, None, 0) is None and fused.layer_norm(x, w).shape == (6, 40)
    a, w = torch.ones(6, 40), torch.ones(40)
    neg = torch.ones(6, 40, dtype=torch.complex64).conj().imag
    assert neg.is_neg() and ext.train_norm(neg, w, None, 1e-6, True) is None
    assert ext.train_norm(a, neg[0], None, 1e-6, True) is None and ext.dropout(a, neg, 9, 1, 1, None) is None
    assert ext.train_norm(torch._efficientzerotensor((3, 40)), w, None, 1e-6, True) is None
    seen = []

    def inside(t):  # t, or a tensor that the transform does not know of
        seen.append(ext.train_norm(t, w, None, 1e-6, True) is None and ext.dropout(a, None, 9, 1, 1, None) is None)
        return t.sum()
    torch.func.vmap(inside)(a)
    torch.func.grad(inside)(a)
    torch.func.jvp(inside, (a,), (a,))
    make_fx(inside)(a)
    torch.jit.trace(inside, (a,), check_trace=False)
    assert len(seen) == 5 and all(seen)
    with pytest.raises(RuntimeError, match="CUDA"):  # and outside of all that they are refused where they are
        ext.train_norm(a, w, None, 1e-6, True)


def test_fake_tensors_take_the_plain_forms_of_the_student_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(2, 6, 256, dtype=BF, device="cuda"), torch.empty(256, device="cuda")
        cw, route = torch.empty(256, 4, device="cuda"), torch.empty(3, 4, dtype=torch.int64, device="cuda")
        kernels.reset()
        assert fused.rms_norm(x, w, 1e-6).shape == fused.gated_rms_norm(x, x, w, 1e-6).shape == x.shape
        assert fused.conv_silu(x, cw).shape == x.shape and fused.swiglu(x).shape == (2, 6, 128)
        assert fused.moe_combine(x.view(12, 256), route.view(-1), torch.empty(3, 4, device="cuda")).shape == (3, 256)
        assert fused.moe_dispatch(x[0], route.view(-1), route.view(-1), 2) is None
    assert not kernels.counts()["native"]


def test_dual_tensors_never_reach_the_kernels():
    """A tangent would be dropped without an error: a dual tensor does not require a gradient."""
    pytest.importorskip("arc_forge_2026_b200._C")
    import torch.autograd.forward_ad as fwad

    from arc_forge_2026_b200.ops import C
    x, w = torch.ones(6, 40), torch.ones(40)
    with fwad.dual_level():
        xd, wd = fwad.make_dual(x, x), fwad.make_dual(w, w)
        for args in ((xd, w, None), (x, wd, None), (x, w, wd)):
            assert C().train_norm(*args, 1e-6, False) is None
        assert C().dropout(xd, None, 9, 1, 1, None) is None
        assert C().dropout(x, xd, 9, 1, 1, None) is None
