"""The trainers' feed-forward operators on the GPU (gated feed-forward block, trainable norms, counter-based dropout)
against their formulas in fp64.

Tolerances are elementwise bounds. With u the relative half step of the element type and e = 2^-23 the largest
relative error of one fp32 addition (rounded or truncated), a sum of K products computed in any order is off by at most
K e sum |a b|; a value rounded to the element type by u |v|. The bounds below add those up through each formula.
"""
import math

import pytest
import torch

from arc_forge_2026_b200.ops import check_status
from arc_forge_2026_b200.train import fused, kernels
from arc_forge_2026_b200.train.ffn import gated_ffn

pytestmark = pytest.mark.gpu
dev = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -23


def u_of(dt):
    return torch.finfo(dt).eps / 2


def ffn_inputs(T, H, F, N, dt, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)

    def rn(*s, k=1.0):
        return (torch.randn(*s, generator=g) * k).to(dt).to(dev)
    return (rn(T, H), rn(2 * F, H, k=H ** -0.5), rn(N, F, k=F ** -0.5), rn(T, N) if residual else None, rn(T, N))


def act64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def ffn_oracle(x, w13, w2, res, dy, act):
    """{name: (value, bound)} in fp64."""
    u = u_of(x.dtype)
    x, w13, w2, dy = (t.double() for t in (x, w13, w2, dy))
    r = torch.zeros_like(dy) if res is None else res.double()
    F, H, T, N = w2.shape[1], x.shape[1], x.shape[0], w2.shape[0]
    gu, gua = x @ w13.T, x.abs() @ w13.abs().T
    g, up = gu[:, :F], gu[:, F:]
    eg, eu = H * E * gua[:, :F], H * E * gua[:, F:]
    a, da = act64(act, g)
    # the activation itself in fp32: exp / tanh / erf to a few units in 2^-22 of its size or of |g|; |act'|, |act''| <= 1.2
    ea, eda = 1.2 * eg + 16 * E * (a.abs() + g.abs()), 1.2 * eg + 16 * E * (1 + g.abs())
    h = a * up
    eh = u * h.abs() + (ea * (up.abs() + eu) + (a.abs() + ea) * eu) + 4 * E * h.abs()
    y = h @ w2.T + r
    ey = eh @ w2.abs().T + F * E * ((h.abs() + eh) @ w2.abs().T) + 2 * E * r.abs()
    dh = dy @ w2
    edh = N * E * (dy.abs() @ w2.abs())
    dg, du = dh * up * da, dh * a
    edg = edh * (up.abs() + eu) * (da.abs() + eda) + dh.abs() * (eu * (da.abs() + eda) + up.abs() * eda)
    edu = edh * (a.abs() + ea) + dh.abs() * ea
    dgu = torch.cat([dg, du], 1)
    edgu = torch.cat([edg, edu], 1)
    edgu = edgu + (u + 8 * E) * (dgu.abs() + edgu)
    A = dgu.abs() + edgu
    out = {"y": (y, ey), "dx": (dgu @ w13, edgu @ w13.abs() + 2 * F * E * (A @ w13.abs())),
           "dw13": (dgu.T @ x, edgu.T @ x.abs() + T * E * (A.T @ x.abs())),
           "dw2": (dy.T @ h, dy.abs().T @ eh + T * E * (dy.abs().T @ (h.abs() + eh)))}
    tiny = torch.finfo(torch.float16).tiny * 2 if u == u_of(HF) else 0.0  # fp16 results below its normal range
    return {k: (v, e + u * (v.abs() + e) + tiny) for k, (v, e) in out.items()}


def check(got, value, bound, what):
    assert got.shape == value.shape, what
    d = (got.double() - value).abs()
    bad = ~(d <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((d / bound.clamp_min(1e-300)).max()))


def run_ffn(x, w13, w2, res, dy, act):
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w13, w2)]
    r = None if res is None else res.detach().clone().requires_grad_(True)
    y = gated_ffn(*leaves, act=act, residual=r)
    grads = torch.autograd.grad(y, leaves + ([r] if r is not None else []), dy)
    out = {"y": y.detach(), "dx": grads[0], "dw13": grads[1], "dw2": grads[2]}
    if r is not None:
        assert torch.equal(grads[3], dy)
    return out


# rows, hidden, intermediate, outputs: one element of everything, ragged tiles, one past a tile, K tails, wide and thin
FFN_SIZES = [(1, 8, 8, 8), (3, 64, 40, 72), (5, 8, 264, 8), (17, 200, 24, 520), (128, 256, 128, 256),
             (129, 136, 264, 200), (257, 512, 384, 512), (64, 640, 512, 64), (1001, 72, 136, 264), (300, 264, 1032, 16),
             (70, 136, 3592, 72), (2500, 520, 72, 264)]


@pytest.mark.parametrize("size", FFN_SIZES)
@pytest.mark.parametrize("dt", [BF, HF])
def test_gated_ffn_forward_and_gradients(size, dt):
    for i, act in enumerate(("silu", "gelu_tanh", "gelu")):
        t = ffn_inputs(*size, dt, seed=i, residual=i != 1)
        got = run_ffn(*t, act)
        ref = ffn_oracle(*t, act)
        with torch.no_grad():
            y = gated_ffn(*t[:3], act=act, residual=t[3])
        check_status()
        check(y, *ref["y"], ("y without gradients", act))
        for k in got:
            check(got[k], *ref[k], (k, act))


@pytest.mark.parametrize("T", [1, 2, 7, 8, 15, 16, 17, 31, 33, 64, 65, 100, 128, 129, 192, 255, 256, 257])
def test_gated_ffn_row_counts_of_serving(T):
    t = ffn_inputs(T, 1024, 640, 1024, BF, seed=T)
    ref = ffn_oracle(*t, "silu")
    with torch.no_grad():
        y = gated_ffn(*t[:3], residual=t[3])
    check_status()
    check(y, *ref["y"], T)


@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 13, 16, 17, 25, 32])
@pytest.mark.parametrize("size", [(8, 8, 8), (264, 1032, 520), (1024, 2056, 1032), (2048, 2056, 2048), (4104, 4200, 4104)])
def test_gated_ffn_single_tokens(size, T):
    """Few rows, on both sides of where the kernels change (rows and bytes of weights); fp16 and bf16, rows of
    a wider tensor, with and without what the backward pass reads."""
    for dt, act in ((BF, "silu"), (HF, "gelu")):
        x, w13, w2, res, dy = ffn_inputs(T, size[0], size[1], size[2], dt, seed=T)
        wide = torch.full((T, size[0] + 8), float("nan"), dtype=dt, device=dev)
        wide[:, :size[0]] = x
        got = run_ffn(x, w13, w2, res, dy, act)
        for k, (want, bound) in ffn_oracle(x, w13, w2, res, dy, act).items():
            check(got[k], want, bound, k)
        with torch.no_grad():
            assert torch.equal(gated_ffn(wide[:, :size[0]], w13, w2, act=act, residual=res), got["y"])
    check_status()


@pytest.mark.parametrize("size", [(33, 4096, 4200), (64, 4096, 8200), (65, 4096, 4200), (128, 2048, 6512), (129, 1024, 1032),
                                  (250, 1032, 4184), (256, 1024, 8464), (257, 1024, 1032), (384, 2056, 1048),
                                  (385, 1024, 1032)])
def test_gated_ffn_where_the_kernels_change(size):
    """Both sides of where rows and bytes of weights choose another kernel."""
    T, H, F = size
    t = ffn_inputs(T, H, F, H, BF, seed=T)
    got, ref = run_ffn(*t, "silu"), ffn_oracle(*t, "silu")
    for k in got:
        check(got[k], *ref[k], k)
    check_status()


@pytest.mark.parametrize("size", [(64, 4096, 7320), (64, 4096, 7328), (65, 2048, 5688), (128, 2048, 5704), (256, 1024, 4392),
                                  (129, 1024, 4400), (257, 2048, 1784), (384, 2048, 1792), (8, 2048, 6912), (2, 2048, 6920),
                                  (9, 2048, 2192), (16, 2048, 2200)])
def test_gated_ffn_at_the_limits_of_rows_and_bytes(size):
    """One size below and one above each limit of the weights' bytes; without gradients as well."""
    T, H, F = size
    t = ffn_inputs(T, H, F, H, BF, seed=T)
    got, ref = run_ffn(*t, "silu"), ffn_oracle(*t, "silu")
    for k in got:
        check(got[k], *ref[k], k)
    with torch.no_grad():
        assert torch.equal(gated_ffn(*t[:3], residual=t[3]), got["y"])
    check_status()


@pytest.mark.parametrize("size", [(385, 64, 8192, 1024), (400, 64, 4104, 264), (520, 64, 16392, 8)])
def test_gated_ffn_residual_of_a_split_product(size):
    """Few row tiles and a deep down projection: its K is split, and the residual is added where the parts are; rows of
    a wider tensor, and the second kernel runs with it as without it."""
    T, H, F, N = size
    for dt in (BF, HF):
        x, w13, w2, res, dy = ffn_inputs(T, H, F, N, dt, seed=T)
        wide = torch.full((T, N + 24), float("nan"), dtype=dt, device=dev)
        wide[:, 8:8 + N] = res
        ref = ffn_oracle(x, w13, w2, res, dy, "silu")["y"]
        with torch.no_grad():
            for r in (res, wide[:, 8:8 + N]):
                with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
                    y = gated_ffn(x, w13, w2, residual=r)
                    torch.cuda.synchronize()
                assert any("ffn_reduce_kernel" in e.key for e in prof.key_averages())
                check(y, *ref, (dt, r.stride()))
    check_status()


# every kernel for few rows: one row, mma.sync with one, two and four groups of rows, clusters by weights and by rows
TWO_TERMS = [(1, 72, 512), (2, 72, 512), (8, 72, 512), (16, 72, 512), (32, 72, 512), (4, 72, 600000), (16, 72, 192000),
             (32, 72, 49152), (48, 72, 512), (100, 72, 512), (200, 72, 512), (384, 72, 520)]


def two_term_bound(x, w13, w2):
    """y of the block without gradients for few rows, its bound, and y as it would be if h were rounded once. h goes on
    as two terms, so it is off by u^2 |h| (fp16: or half of its smallest step) beside the fp32 errors of ffn_oracle."""
    u, H, F = u_of(x.dtype), x.shape[1], w2.shape[1]
    a64, b64, c64 = x.double(), w13.double(), w2.double()
    gu, gua = a64 @ b64.T, a64.abs() @ b64.abs().T
    g, up, eg, eu = gu[:, :F], gu[:, F:], H * E * gua[:, :F], H * E * gua[:, F:]
    a, _ = act64("silu", g)
    ea = 1.2 * eg + 16 * E * (a.abs() + g.abs())
    h = a * up
    half_step = torch.finfo(HF).smallest_normal * torch.finfo(HF).eps / 2 if x.dtype == HF else 0.0
    eh = u * u * h.abs() + half_step + (ea * (up.abs() + eu) + (a.abs() + ea) * eu) + 4 * E * h.abs()
    y = h @ c64.T
    e = eh @ c64.abs().T + F * E * ((h.abs() + eh) @ c64.abs().T)
    tiny = torch.finfo(HF).tiny if x.dtype == HF else 0.0
    return y, e + u * (y.abs() + e) + tiny, (h.to(x.dtype).double() @ c64.T).to(x.dtype)


@pytest.mark.parametrize("size", TWO_TERMS)
@pytest.mark.parametrize("dt", [BF, HF])
def test_gated_ffn_keeps_both_terms_of_h_for_few_rows(size, dt):
    T, F, N = size
    x, w13, w2, _, _ = ffn_inputs(T, 8, F, N, dt, seed=T, residual=False)
    y, bound, once = two_term_bound(x, w13, w2)
    assert ((once.double() - y).abs() > bound).any()  # the bound tells the two apart
    with torch.no_grad():
        check(gated_ffn(x, w13, w2), y, bound, size)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    check(gated_ffn(*leaves).detach(), y, bound, "with gradients")
    check_status()


def test_gated_ffn_gradient_against_differences():
    """<gradient, direction> of the kernels against the central difference of the fp64 block along the direction."""
    x, w13, w2, res, dy = ffn_inputs(96, 128, 200, 64, BF, seed=3)
    got = run_ffn(x, w13, w2, res, dy, "silu")
    ref = ffn_oracle(x, w13, w2, res, dy, "silu")
    g = torch.Generator().manual_seed(9)

    def loss(x, w13, w2):
        gu = x @ w13.T
        a, _ = act64("silu", gu[:, :200])
        return ((a * gu[:, 200:]) @ w2.T * dy.double()).sum()
    base = [t.double() for t in (x, w13, w2)]
    for i, name in enumerate(("dx", "dw13", "dw2")):
        v = torch.randn(base[i].shape, generator=g, dtype=torch.float64).to(dev)
        eps = 1e-5
        lo, hi = list(base), list(base)
        lo[i], hi[i] = base[i] - eps * v, base[i] + eps * v
        num = (loss(*hi) - loss(*lo)) / (2 * eps)
        bound = (ref[name][1] * v.abs()).sum() + 1e-6 * num.abs() + 1e-6 * (ref[name][0].abs() * v.abs()).sum()
        assert (num - (got[name].double() * v).sum()).abs() <= bound, name


def test_gated_ffn_strides_and_gradient_subsets():
    T, H, F, N = 70, 136, 72, 40
    x, w13, w2, res, dy = ffn_inputs(T, H, F, N, BF, seed=4)
    ref = ffn_oracle(x, w13, w2, res, dy, "silu")
    wide = torch.zeros(T, H + 24, dtype=BF, device=dev)
    wide[:, 8:8 + H] = x                                    # a strided view with an aligned base
    odd = torch.zeros(T * H + 3, dtype=BF, device=dev)
    odd[3:] = x.reshape(-1)                                 # a base no tensor map can start at
    tr = x.t().contiguous().t()                             # column-major rows
    for xv in (wide[:, 8:8 + H], odd[3:].view(T, H), tr):
        leaf = xv.detach().requires_grad_(True)
        w13t = w13.t().contiguous().t().requires_grad_(True)
        y = gated_ffn(leaf, w13t, w2, residual=res.t().contiguous().t())
        dx, dw13 = torch.autograd.grad(y, [leaf, w13t], dy.t().contiguous().t())
        check(y.detach(), *ref["y"], "y")
        check(dx, *ref["dx"], "dx")
        check(dw13, *ref["dw13"], "dw13")
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        ls = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, w13, w2), need)]
        y = gated_ffn(*ls, residual=res)
        gs = torch.autograd.grad(y, [t for t in ls if t.requires_grad], dy)
        for name, gr in zip([n for n, k in zip(("dx", "dw13", "dw2"), need) if k], gs):
            check(gr, *ref[name], (need, name))
    # leading dimensions, and a gradient broadcast from a scalar
    x3 = x.view(7, 10, H).clone().requires_grad_(True)
    gated_ffn(x3, w13, w2).sum().backward()
    one = ffn_oracle(x, w13, w2, None, torch.ones_like(dy), "silu")
    check(x3.grad.view(T, H), *one["dx"], "dx of a sum")
    check_status()


def test_gated_ffn_no_rows_and_bad_values():
    x, w13, w2, res, dy = ffn_inputs(0, 64, 32, 48, BF)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    y = gated_ffn(*leaves)
    assert y.shape == (0, 48)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, torch.empty(0, 48, dtype=BF, device=dev))
    assert dx.shape == (0, 64) and not dw13.any() and not dw2.any()
    # a NaN or an infinity stays in its row of y and dx
    x, w13, w2, res, dy = ffn_inputs(200, 64, 32, 48, BF, seed=5)
    x[3, 5], x[150, 0] = float("nan"), float("inf")
    got = run_ffn(x, w13, w2, None, dy, "silu")
    rest = torch.ones(200, dtype=torch.bool)
    rest[3] = rest[150] = False
    assert torch.isfinite(got["y"][rest]).all() and torch.isfinite(got["dx"][rest]).all()
    assert torch.isnan(got["y"][3]).all()
    check_status()


@pytest.mark.parametrize("T", [1, 4, 30, 100, 500])
def test_gated_ffn_fp16_range_of_the_intermediate_row(T):
    """An h past fp16's largest number is infinite, in its own row alone; just below it everything is finite. bf16 has
    the range of fp32."""
    for dt, scale, finite in ((HF, 1.01, False), (HF, 0.99, True), (BF, 100.0, True)):
        x, w13, w2 = (torch.zeros(*s, dtype=dt, device=dev) for s in ((T, 8), (16, 8), (16, 8)))
        x[:, 0], x[:, 1] = 16, 16
        w13[0, 0] = w13[8, 1] = 8  # g = u = 128: h = 16,384, silu(128) being 128
        w2[:, 0] = 2.0 ** -6       # y = 256
        big = (T - 1) // 2
        x[big, 1] = 64 * scale     # h = 65,536 x scale, and 65,504 is the largest
        with torch.no_grad():
            y = gated_ffn(x, w13, w2)
        rest = [i for i in range(T) if i != big]
        assert (y[rest] == 256).all()
        if finite:
            h = float(x[big, 1]) * 8 * 128
            assert ((y[big].double() - h / 64).abs() <= 3 * u_of(dt) * h / 64).all()
        else:
            assert not torch.isfinite(y[big]).any()
    check_status()


def test_gated_ffn_repeats_bitwise_and_on_other_streams():
    t = ffn_inputs(333, 256, 136, 256, BF, seed=6)
    a = run_ffn(*t, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = run_ffn(*t, "silu")
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for k in a:
        assert torch.equal(a[k], b[k]), k


def test_feed_forward_half_layer_captured_and_replayed():
    """norm -> gated block -> dropout + residual, forward and backward, in two graphs that are replayed in turn with
    new inputs and new random offsets; each replay equals the eager call."""
    T, H, F = 130, 256, 136
    _, w13, w2, _, _ = ffn_inputs(T, H, F, H, BF, seed=7)
    g = torch.Generator().manual_seed(8)
    nw = (1 + 0.1 * torch.randn(H, generator=g)).to(dev)
    nb = (0.1 * torch.randn(H, generator=g)).to(dev)

    def step(x, params, dy, rng):
        y = fused.layer_norm(x, params[2], params[3], 1e-6)
        y = gated_ffn(y, params[0], params[1])
        y = fused.dropout(y, 0.25, rng, residual=x)
        return [y] + list(torch.autograd.grad(y, [x, *params], dy))
    data = [[(torch.randn(T, H, generator=g).to(BF).to(dev), torch.randn(T, H, generator=g).to(BF).to(dev),
              torch.tensor([5 + i, 1000 * i], device=dev)) for i in range(3)] for _ in range(2)]
    graphs = []
    for _ in range(2):
        x = torch.zeros(T, H, dtype=BF, device=dev).requires_grad_(True)
        dy, rng = torch.zeros(T, H, dtype=BF, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
        params = [t.detach().clone().requires_grad_(True) for t in (w13, w2, nw, nb)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(x, params, dy, rng)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(x, params, dy, rng)
        graphs.append((gr, x, dy, rng, out))
    for i in range(3):
        for k, (gr, x, dy, rng, out) in enumerate(graphs):
            with torch.no_grad():
                x.copy_(data[k][i][0])
                dy.copy_(data[k][i][1])
                rng.copy_(data[k][i][2])
            gr.replay()
        torch.cuda.synchronize()
        for k, (gr, x, dy, rng, out) in enumerate(graphs):
            params = [t.detach().clone().requires_grad_(True) for t in (w13, w2, nw, nb)]
            ref = step(data[k][i][0].clone().requires_grad_(True), params, data[k][i][1], data[k][i][2])
            for a, b in zip(out, ref):
                assert torch.equal(a, b), (i, k)
    check_status()


# ------------------------------------------------------------------------------------------------------------- norms
def norm_oracle(x, w, b, dy, eps, rms):
    u, uw = u_of(x.dtype), u_of(w.dtype)
    W, T = x.shape[-1], x.shape[0]
    x, w, dy = x.double(), w.double(), dy.double()
    depth = 64  # additions an element goes through in a row sum: 32 of its lane, 5 of the warp, 16 of the row's warps
    mean = torch.zeros_like(x[:, :1]) if rms else x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = (xc.square().mean(-1, keepdim=True) + eps).rsqrt()
    ec = 0 * x if rms else E * (x.abs() + 2 * depth * x.abs().mean(-1, keepdim=True))
    # relative error of rstd: half that of the mean square (its sum, and the errors of xc in it), and rsqrtf
    er = depth * E + (ec * xc.abs()).mean(-1, keepdim=True) * rstd.square() + (ec * ec).mean(-1, keepdim=True) * rstd.square()
    xh = xc * rstd
    eh = ec * rstd + xh.abs() * (er + 4 * E)
    m = 1 + w if rms else w
    bb = torch.zeros_like(w) if b is None else b.double()
    y = xh * m + bb
    ey = eh * m.abs() + 4 * E * ((xh * m).abs() + bb.abs())
    v = dy * m
    ev = 2 * E * v.abs()
    m1 = (v * xh).mean(-1, keepdim=True)
    em1 = (depth * E * (v * xh).abs() + ev * xh.abs() + v.abs() * eh).mean(-1, keepdim=True)
    m0 = torch.zeros_like(m1) if rms else v.mean(-1, keepdim=True)
    em0 = (depth * E * v.abs() + ev).mean(-1, keepdim=True)
    dx = rstd * (v - m0 - xh * m1)
    edx = rstd * (ev + em0 + eh * m1.abs() + xh.abs() * em1 + 4 * E * (v.abs() + m0.abs() + (xh * m1).abs())) \
        + dx.abs() * (er + 4 * E)
    dw, edw = (dy * xh).sum(0), (dy.abs() * eh).sum(0) + (T + 8) * E * (dy * xh).abs().sum(0)
    db, edb = dy.sum(0), (T + 8) * E * dy.abs().sum(0)
    tiny = torch.finfo(HF).tiny
    return {"y": (y, ey + u * (y.abs() + ey) + tiny), "dx": (dx, edx + u * (dx.abs() + edx) + tiny),
            "dw": (dw, edw + uw * (dw.abs() + edw) + tiny), "db": (db, edb + uw * (db.abs() + edb) + tiny)}


def norm_inputs(T, W, dt, wdt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, W, generator=g) + 0.5) * torch.exp(torch.randn(T, 1, generator=g))
    return (x.to(dt).to(dev), (1 + 0.2 * torch.randn(W, generator=g)).to(wdt).to(dev),
            (0.2 * torch.randn(W, generator=g)).to(wdt).to(dev), torch.randn(T, W, generator=g).to(dt).to(dev))


def run_norm(x, w, b, dy, eps, rms):
    ls = [t.detach().requires_grad_(True) for t in ([x, w] if rms or b is None else [x, w, b])]
    y = fused.rms_norm(ls[0], ls[1], eps) if rms else fused.layer_norm(ls[0], ls[1], ls[2] if b is not None else None, eps)
    gs = torch.autograd.grad(y, ls, dy)
    return dict(zip(("y", "dx", "dw", "db"), (y.detach(), *gs)))


@pytest.mark.parametrize("W", [1, 7, 8, 33, 128, 256, 264, 768, 1001, 1002, 1024, 1152, 1160, 2048, 2056, 2560, 4095,
                               4606, 4608, 5000, 8192, 8200, 16384])
@pytest.mark.parametrize("rms", [False, True])
def test_trainable_norms(W, rms):
    for i, (dt, wdt, T) in enumerate([(BF, FP, 37), (BF, BF, 700), (HF, HF, 5), (HF, FP, 1), (FP, FP, 300)]):
        x, w, b, dy = norm_inputs(T, W, dt, wdt, seed=i)
        b = None if i == 2 else b
        got = run_norm(x, w, b, dy, 1e-6, rms)
        ref = norm_oracle(x, w, None if rms else b, dy, 1e-6, rms)
        for k in got:
            check(got[k], *ref[k], (k, dt, wdt, T))


@pytest.mark.parametrize("W", [2816, 3201, 3202, 3208, 3848, 4088, 4096, 4104, 4616])
def test_trainable_norms_where_the_chunks_of_a_lane_change(W):
    """Two and three chunks a lane in the backward pass; rows by eight, by pairs and one by one."""
    for i, (dt, wdt, T, rms) in enumerate([(BF, FP, 37, False), (BF, BF, 700, True), (HF, FP, 1, False), (FP, FP, 300, False)]):
        x, w, b, dy = norm_inputs(T, W, dt, wdt, seed=i)
        got = run_norm(x, w, b, dy, 1e-6, rms)
        ref = norm_oracle(x, w, None if rms else b, dy, 1e-6, rms)
        for k in got:
            check(got[k], *ref[k], (k, dt, wdt, T))
    check_status()


def test_norm_strides_empty_frozen_and_constant_rows():
    x, w, b, dy = norm_inputs(50, 264, BF, FP, seed=11)
    ref = norm_oracle(x, w, b, dy, 1e-6, False)
    wide = torch.zeros(50, 304, dtype=BF, device=dev)
    for off in (8, 2, 3):  # views whose rows start on 16 bytes, on 4 and on 2
        wide[:, off:off + 264] = x
        got = run_norm(wide[:, off:off + 264], w, b, dy.t().contiguous().t(), 1e-6, False)
        for k in got:
            check(got[k], *ref[k], (k, off))
    x0 = torch.empty(0, 264, dtype=BF, device=dev)
    got = run_norm(x0, w, b, x0, 1e-6, False)
    assert got["dx"].shape == (0, 264) and not got["dw"].any() and not got["db"].any()
    # only x, only w, only b
    for i, k in enumerate(("dx", "dw", "db")):
        ls = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        (gr,) = torch.autograd.grad(fused.layer_norm(*ls, 1e-6), [ls[i]], dy)
        check(gr, *ref[k], k)
    # constant rows: the variance is 0 and y is the bias
    c = torch.full((3, 264), 7.0, dtype=BF, device=dev)
    assert torch.equal(fused.layer_norm(c, w, b, 1e-6), b.to(BF).expand(3, -1))
    # leading dimensions
    y = fused.layer_norm(x.view(5, 10, 264), w, b, 1e-6)
    assert torch.equal(y.view(50, 264), fused.layer_norm(x, w, b, 1e-6))
    # a frozen weight at the model's widths stays on the student's kernel, bit for bit
    xs = norm_inputs(9, 2048, BF, FP, seed=12)[0]
    ws = torch.randn(2048, device=dev) * 0.1
    y = torch.empty_like(xs)
    from arc_forge_2026_b200.ops import C
    C().rmsnorm_train(xs, None, ws, 1e-6, y, torch.empty(9, device=dev), None, None, None)
    assert torch.equal(y, fused.rms_norm(xs, ws, 1e-6))


@pytest.mark.parametrize("W", [2, 264, 1002, 1152, 4608, 8200])
@pytest.mark.parametrize("dt", [BF, HF])
def test_norm_weights_at_any_element_of_a_flat_buffer(W, dt):
    """16-bit w and b as views that start 2, 4, 6 or 16 bytes into a buffer, w and b each for itself."""
    x, w, b, dy = norm_inputs(40, W, dt, dt, seed=15)

    def at(t, off):
        buf = torch.zeros(W + 16, dtype=dt, device=dev)
        buf[off:off + W] = t
        return buf[off:off + W]
    for rms in (False, True):
        ref = norm_oracle(x, w, None if rms else b, dy, 1e-6, rms)
        for ow, ob in ((1, 0), (0, 1), (2, 0), (0, 2), (3, 5), (8, 2), (8, 8)):
            got = run_norm(x, at(w, ow), at(b, ob), dy, 1e-6, rms)
            for k in got:
                check(got[k], *ref[k], (k, rms, ow, ob))
    check_status()


def test_norm_repeats_bitwise():
    x, w, b, dy = norm_inputs(3001, 1152, BF, FP, seed=13)
    a, c = run_norm(x, w, b, dy, 1e-6, False), run_norm(x, w, b, dy, 1e-6, False)
    for k in a:
        assert torch.equal(a[k], c[k]), k


def test_many_rows_pass_32_bit_offsets():
    """More than 2^31 elements: the last rows equal those of a small call."""
    rows, W = (1 << 31) // 1024 + 9, 1024
    x = torch.zeros(rows, W, dtype=BF, device=dev)
    tail = norm_inputs(9, W, BF, FP, seed=14)
    x[-9:] = tail[0]
    y = fused.layer_norm(x, tail[1], tail[2], 1e-6)
    assert torch.equal(y[-9:], fused.layer_norm(tail[0], tail[1], tail[2], 1e-6))
    del y
    z = fused.dropout(x, 0.5, 3, 0)
    off = (rows - 9) * W // 8
    assert torch.equal(z[-9:], fused.dropout(tail[0], 0.5, 3, off))


# ----------------------------------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (37, 1001), (64, 256), (2, 3, 40)])
@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_dropout_equals_its_definition(shape, dt):
    g = torch.Generator().manual_seed(1)
    x, r, dy = (torch.randn(*shape, generator=g).to(dt) for _ in range(3))
    for p, seed, off in ((0.0, 1, 0), (0.1, 2 ** 63 + 17, 2 ** 32 - 2), (0.5, -5, 2 ** 40), (0.999, 7, 1), (1.0, 7, 1)):
        for res in (None, r):
            lx = x.to(dev).requires_grad_(True)
            lr = None if res is None else r.to(dev).requires_grad_(True)
            y = fused.dropout(lx, p, seed, off, residual=lr)
            gs = torch.autograd.grad(y, [lx] + ([] if lr is None else [lr]), dy.to(dev))
            # the scale is one fp32 number on both sides, one product and one sum are rounded once each
            assert torch.equal(y.cpu(), fused.dropout(x, p, seed, off, residual=res)), (p, seed)
            assert torch.equal(gs[0].cpu(), fused.dropout(dy, p, seed, off))
            assert lr is None or torch.equal(gs[1].cpu(), dy)


def test_dropout_views_bad_values_seed_tensors_and_streams():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, 50, generator=g).to(BF).to(dev)
    want = fused.dropout(x, 0.3, 11, 5)
    buf = torch.zeros(2001, dtype=BF, device=dev)
    buf[1:] = x.reshape(-1)
    assert torch.equal(fused.dropout(buf[1:].view(40, 50), 0.3, 11, 5), want)          # unaligned base
    assert torch.equal(fused.dropout(x.t().contiguous().t(), 0.3, 11, 5), want)        # logical order, not memory's
    assert torch.equal(fused.dropout(x, 0.3, torch.tensor([11, 5], device=dev)), want)
    assert torch.equal(fused.dropout(x, 0.3, torch.tensor([11, 2], device=dev), 3), want)
    assert not torch.equal(fused.dropout(x, 0.3, 11, 6), want)
    bad = x.clone()
    dropped = want == 0
    bad[dropped] = float("nan")
    assert torch.equal(fused.dropout(bad, 0.3, 11, 5), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = fused.dropout(x, 0.3, 11, 5)
    s.synchronize()
    assert torch.equal(other, want)
    # a seed tensor changed between forward and backward is refused, not silently another mask
    rng = torch.tensor([1, 2], device=dev)
    y = fused.dropout(x.clone().requires_grad_(True), 0.3, rng)
    rng.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert fused.dropout(torch.empty(0, 4, dtype=BF, device=dev), 0.3, 1).shape == (0, 4)


def test_registry_counts_the_native_calls():
    kernels.reset()
    x, w, b, dy = norm_inputs(4, 64, BF, FP)
    fused.layer_norm(x, w, b)
    fused.rms_norm(x, w.requires_grad_(True), 1e-6)
    fused.dropout(x, 0.1, 1)
    c = kernels.counts()
    assert c["native"] == {"layer_norm": 1, "rms_norm": 1, "dropout": 1} and not c["fallback"]


def _with_opt_in(fn):
    old = {n for n in kernels.NAMES if kernels.enabled(n)}
    try:
        kernels.enable(sorted(old | {"gated_ffn"}))
        kernels.reset()
        return fn(), kernels.counts()
    finally:
        kernels.enable(sorted(old))


def test_student_and_drafter_take_the_block_when_asked():
    """The opt-in path against the default one: the same products with other roundings. Each side rounds the
    intermediate values of one layer's shared expert a few times, so the results agree to a few bf16 half steps."""
    from arc_forge_2026_b200.config import drafter_preset, preset
    from arc_forge_2026_b200.train.drafter_train import DrafterTrain
    from arc_forge_2026_b200.train.student import random_student
    st = random_student(preset("tiny_gpu"), dev, seed=0, checkpoint_layers=False)
    moe = st.layers[0].moe
    x = torch.randn(130, st.cfg.hidden_size, generator=torch.Generator().manual_seed(1)).to(BF).to(dev)

    def step():
        lx = x.clone().requires_grad_(True)
        y = moe(lx)
        return [y.detach(), *torch.autograd.grad(y.float().square().sum(), [lx, moe.shared_w13, moe.shared_down])]
    base = step()
    got, counts = _with_opt_in(step)
    assert counts["native"]["gated_ffn"] == 1 and not counts["fallback"].get("gated_ffn")
    for a, b in zip(got, base):
        assert a.dtype == b.dtype and ((a - b).float().norm() / b.float().norm()) < 4 * u_of(BF)
    cfg = drafter_preset("tiny")
    dt = DrafterTrain(cfg, 256, 512, torch.arange(128), device=dev)
    m, y = dt.layers[0], torch.randn(6, cfg.k, cfg.hidden_size, device=dev)

    def dstep():
        o = dt._ffn(m, y, 0, None)
        return [o.detach(), *torch.autograd.grad(o.square().sum(), [m.w13, m.w2])]
    base = dstep()
    got, counts = _with_opt_in(dstep)
    assert counts["native"]["gated_ffn"] == 1
    for a, b in zip(got, base):  # fp32 products against bf16 operands: three rounded factors a product
        assert a.dtype == FP and ((a - b).norm() / b.norm()) < 6 * u_of(BF)
    check_status()


def test_drafter_with_a_shared_feed_forward_takes_the_block_twice():
    """Dense and shared feed-forward of a dense_shared drafter, bf16 operands against fp32 products: each part and each
    weight gradient of a linear loss is off by three rounded factors a product, as above."""
    from arc_forge_2026_b200.config import drafter_preset
    from arc_forge_2026_b200.train.drafter_train import DrafterTrain
    cfg = drafter_preset("tiny", ffn="dense_shared", shared_intermediate_size=64)
    dt = DrafterTrain(cfg, 256, 512, torch.arange(128), device=dev)
    m = dt.layers[0]
    g = torch.Generator(device=dev).manual_seed(4)
    y, v = (torch.randn(6, cfg.k, cfg.hidden_size, device=dev, generator=g) for _ in range(2))

    def step():
        o = dt._ffn(m, y, 0, None)
        return [o.detach(), *torch.autograd.grad((o * v).sum(), [m.w13, m.w2, m.sw13, m.sw2])]
    base = step()
    dense, shared = dt._gated(y, m.w13, m.w2), torch.sigmoid(y @ m.shared_gate.t()) * dt._gated(y, m.sw13, m.sw2)
    got, counts = _with_opt_in(step)
    assert counts["native"]["gated_ffn"] == 2 and not counts["fallback"].get("gated_ffn")
    assert (got[0] - base[0]).norm() <= 6 * u_of(BF) * (dense.norm() + shared.norm())
    for a, b in zip(got[1:], base[1:]):
        assert a.dtype == FP and (a - b).norm() <= 6 * u_of(BF) * b.norm()
    check_status()


def test_lora_dropout_on_the_native_products():
    """An adapter's output and gradients with dropout equal those of the adapter without it on the dropped input."""
    from arc_forge_2026_b200.train.lora import LoRAAdapter
    g = torch.Generator(device=dev).manual_seed(2)
    ad = LoRAAdapter(256, 128, 16, 32.0, dev, g, dropout=0.2, dropout_seed=9)
    with torch.no_grad():
        ad.B.normal_(generator=g)
    ad.dropout_step = 3
    x = torch.randn(200, 256, generator=g, device=dev).to(BF).requires_grad_(True)
    y = ad(x)
    dx, dA, dB = torch.autograd.grad(y.square().sum(), [x, ad.A, ad.B])
    ad.eval()
    xd = fused.dropout(x.detach(), 0.2, 9, 3 << 36).requires_grad_(True)
    y2 = ad(xd)
    dx2, dA2, dB2 = torch.autograd.grad(y2.square().sum(), [xd, ad.A, ad.B])
    assert torch.equal(y, y2) and torch.equal(dA, dA2) and torch.equal(dB, dB2)
    assert torch.equal(dx, fused.dropout(dx2, 0.2, 9, 3 << 36))


def test_checkpointed_student_layer_and_second_derivatives():
    """Activation checkpointing recomputes the same values (dropout masks among them) through the C++ autograd nodes;
    create_graph is refused where it would give second derivatives that lack terms."""
    from arc_forge_2026_b200.config import preset
    from arc_forge_2026_b200.train import lora
    from arc_forge_2026_b200.train.student import random_student
    ids = torch.randint(0, 200, (1, 192), generator=torch.Generator().manual_seed(3)).to(dev)

    def grads(ckpt):
        st = random_student(preset("tiny_gpu"), dev, seed=0, checkpoint_layers=ckpt)
        ps = lora.attach_lora(st, 16, 16.0, seed=1, dropout=0.25)
        with torch.no_grad():
            for i, p in enumerate(ps):
                p.add_(torch.randn(p.shape, generator=torch.Generator().manual_seed(i)).to(dev) * 0.05)
        lora.set_dropout_step(st, 4)
        return torch.autograd.grad(st.hidden(ids).float().square().sum(), ps)
    (a, ca), (b, cb) = _with_opt_in(lambda: grads(True)), _with_opt_in(lambda: grads(False))
    assert ca["native"]["gated_ffn"] > cb["native"]["gated_ffn"] > 0 and ca["native"]["dropout"] > 0
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    x, w13, w2, res, dy = ffn_inputs(8, 16, 8, 16, BF)
    for f in (lambda t: gated_ffn(t, w13, w2), lambda t: fused.dropout(t, 0.5, 1)):
        leaf = x.clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(f(leaf).float().sum(), leaf, create_graph=True)


def test_gpu_refusals():
    x, w13, w2, res, dy = ffn_inputs(8, 16, 8, 16, BF)
    for kw in (dict(act="relu"), dict(w2=w2[:, :4]), dict(w2=w2.float()), dict(w13=w13.cpu()), dict(residual=res[:4]),
               dict(residual=res.float())):
        with pytest.raises(ValueError):
            gated_ffn(**{**dict(x=x, w13=w13, w2=w2), **kw})
    with pytest.raises(ValueError):
        fused.layer_norm(x, torch.ones(15, device=dev))
    with pytest.raises(ValueError):
        fused.layer_norm(x, torch.ones(16))
    with pytest.raises(ValueError):
        fused.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    # outside what the kernels take: the plain form, counted as such where the registry counts
    y = gated_ffn(x[:, :12], w13[:, :12], w2)
    assert y.shape == (8, 16)
    wide = torch.randn(2, 16392, device=dev)
    kernels.reset()
    y = fused.layer_norm(wide, torch.ones(16392, device=dev), None, 1e-6)
    assert kernels.counts()["fallback"] == {"layer_norm": 1}
    check(y, *norm_oracle(wide, torch.ones(16392, device=dev), None, wide, 1e-6, False)["y"], "wide")
    z = torch.randn(4, 16, dtype=torch.float64, device=dev)
    assert torch.equal(fused.dropout(z, 0.5, 3).cpu(), fused.dropout(z.cpu(), 0.5, 3))


def test_results_can_be_changed_in_place_and_graphs_walked_twice():
    x, w13, w2, res, dy = ffn_inputs(24, 32, 16, 32, BF, seed=20)
    nw = torch.ones(32, device=dev, dtype=BF)
    for f in (lambda t: gated_ffn(t, w13, w2), lambda t: fused.layer_norm(t, nw), lambda t: fused.rms_norm(t, nw, 1e-6),
              lambda t: fused.dropout(t, 0.3, 4)):
        for shape in ((24, 32), (2, 3, 4, 32)):
            leaf = x.view(shape).clone().requires_grad_(True)
            y = f(leaf)
            y += 1
            y.mul_(2)
            (a,) = torch.autograd.grad(y, leaf, dy.view(y.shape), retain_graph=True)
            (b,) = torch.autograd.grad(y, leaf, dy.view(y.shape))
            assert torch.equal(a, b)
            (c,) = torch.autograd.grad(f(leaf), leaf, 2 * dy.view(y.shape))
            assert torch.equal(a, c)
    # a saved input changed in place before the backward pass is refused
    leaf = x.clone().requires_grad_(True)
    z = leaf * 1
    y = gated_ffn(z, w13, w2)
    z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_single_vectors_and_broadcast_rows():
    """1-D inputs are one row; an expanded input (row stride 0) gives the gradient of the row it repeats."""
    x, w13, w2, res, dy = ffn_inputs(9, 64, 24, 40, BF, seed=21)
    w = (1 + 0.1 * torch.randn(64, generator=torch.Generator().manual_seed(1))).to(dev)
    assert torch.equal(gated_ffn(x[0], w13, w2), gated_ffn(x[:1], w13, w2)[0])
    assert torch.equal(fused.layer_norm(x[0], w), fused.layer_norm(x[:1], w)[0])
    one = x[:1].clone().requires_grad_(True)
    rows = one.expand(9, 64)
    dn = torch.randn(9, 64, generator=torch.Generator().manual_seed(2)).to(BF).to(dev)
    full = x[:1].repeat(9, 1).requires_grad_(True)
    for f, d in ((lambda t: gated_ffn(t, w13, w2), dy), (lambda t: fused.layer_norm(t, w), dn)):
        (a,) = torch.autograd.grad(f(rows), one, d, retain_graph=True)
        (b,) = torch.autograd.grad(f(full), full, d)
        assert torch.equal(a, b.sum(0, keepdim=True, dtype=BF))
    check_status()


@pytest.mark.parametrize("rms", [False, True])
def test_norm_second_derivatives(rms):
    """create_graph through the norms: the second derivatives equal autograd's of the plain form in fp64."""
    g = torch.Generator().manual_seed(21)
    x, w, b, dy, k = (torch.randn(*s, generator=g).to(dev) for s in ((6, 40), (40,), (40,), (6, 40), (6, 40)))

    def second(f, *ts):
        ls = [t.clone().requires_grad_(True) for t in ts]
        y = f(*ls)
        first = torch.autograd.grad(y, ls, dy.to(y.dtype), create_graph=True)
        return [*first, *torch.autograd.grad((first[0] * k.to(y.dtype)).sum() + first[1].square().sum(), ls[:2])]

    def plain(x, w, *b):
        c = x if rms else x - x.mean(-1, keepdim=True)
        y = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-5) * (1 + w if rms else w)
        return y if rms else y + b[0]
    ts = (x, w) if rms else (x, w, b)
    got = second((lambda x, w: fused.rms_norm(x, w, 1e-5)) if rms else (lambda x, w, b: fused.layer_norm(x, w, b)), *ts)
    want = second(plain, *(t.double() for t in ts))
    for a, r in zip(got, want):
        # sums of at most 40 x 6 terms, each the product of a few fp32 values; inputs and derivatives of order 1 to 100
        assert (a.double() - r).abs().max() <= 2 * 240 * E * max(1.0, float(r.detach().abs().max())) * 4


def test_backward_captured_while_an_eager_graph_of_the_leaves_lives_is_refused():
    """The accumulators of the living graph are on the default stream, which may not join a capture."""
    x, w13, w2, _, dy = ffn_inputs(40, 64, 32, 64, BF, seed=9)
    w = torch.ones(64, device=dev)
    calls = ((lambda x, a, b, w: gated_ffn(x, a, b)), (lambda x, a, b, w: fused.layer_norm(x, w)),
             (lambda x, a, b, w: fused.dropout(x, 0.5, 1)))
    for f in calls:
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w13, w2, w)]
        alive = f(*leaves)  # noqa: F841
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="release that graph first"):
            with torch.cuda.graph(gr):
                f(*leaves).backward(dy)
        torch.cuda.synchronize()
        del alive
        for t in leaves:
            assert t.grad is None
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f(*leaves).backward(dy)
        gr.replay()
        ref = [t.detach().clone().requires_grad_(True) for t in leaves]
        f(*ref).backward(dy)
        for a, r in zip(leaves, ref):
            assert (a.grad is None) == (r.grad is None) and (r.grad is None or torch.equal(a.grad, r.grad))
    check_status()


def test_calls_on_two_streams_at_once():
    """Workspaces belong to a call: the same operators, run on two streams at the same time, give what they give alone."""
    def work(t, w):
        out = []
        for i in range(4):
            out += run_ffn(*t, "silu").values()
            leaf = t[0].clone().requires_grad_(True)
            y = fused.dropout(fused.rms_norm(leaf, w, 1e-6), 0.3, i)
            out += [y, *torch.autograd.grad(y, leaf, t[0])]
        return out
    data = [(ffn_inputs(T, 256, 264, 256, BF, seed=T), torch.randn(256, device=dev).requires_grad_(True))
            for T in (1500, 90)]
    alone = [work(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    both = []
    for d, s in zip(data, streams):
        with torch.cuda.stream(s):
            both.append(work(*d))
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        for u, v in zip(a, b):
            assert torch.equal(u, v)
    check_status()


def _transform_cases():
    """name -> (function of x, inputs, their {name: (value, bound)} from the fp64 formulas, which takes (x, dy))."""
    x, w, b, dy = norm_inputs(12, 264, FP, FP, seed=30)
    keep = fused.dropout_keep_reference(12 * 264, 0.25, 5, 0, dev).view(12, 264).double() * (65536 / 49152)
    fx, w13, w2, _, fdy = ffn_inputs(12, 64, 40, 72, BF, seed=31)

    def drop64(x, dy):  # one rounded scale, one rounded product
        return {n: (t.double() * keep, 4 * E * t.double().abs()) for n, t in (("y", x), ("dx", dy))}
    return {"rms": (lambda t: fused.rms_norm(t, w, 1e-6), x, dy, lambda x, dy: norm_oracle(x, w, None, dy, 1e-6, True)),
            "layer": (lambda t: fused.layer_norm(t, w, b, 1e-6), x, dy,
                      lambda x, dy: norm_oracle(x, w, b, dy, 1e-6, False)),
            "dropout": (lambda t: fused.dropout(t, 0.25, 5), x, dy, drop64),
            "ffn": (lambda t: gated_ffn(t, w13, w2), fx, fdy, lambda x, dy: ffn_oracle(x, w13, w2, None, dy, "silu"))}


def check_tangent(tangent, t, y, dy, dx):
    """<dy, J t> = <J^T dy, t>: the tangent, off by at most as much as dx is (the same factors, in fp32) and one
    rounding."""
    a, b = (dy.double() * tangent.double()).sum(), (dx[0] * t.double()).sum()
    bound = 2 * (dx[1] * t.double().abs()).sum() + 2 * u_of(y.dtype) * (dy.double() * tangent.double()).abs().sum()
    assert tangent.dtype == y.dtype and (a - b).abs() <= bound


@pytest.mark.parametrize("name", ["rms", "layer", "dropout", "ffn"])
def test_function_transforms_and_traces(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x, dy, oracle = _transform_cases()[name]
    ref = oracle(x, dy)
    if name != "dropout":  # (a sample's mask there is that of a tensor of the sample's shape)
        check(torch.func.vmap(f)(x.view(3, 4, -1)).view_as(dy), *ref["y"], "vmap")
    else:
        y = torch.func.vmap(f)(x.view(3, 4, -1))
        assert all(torch.equal(y[i], f(x.view(3, 4, -1)[i])) for i in range(3))
    check(torch.func.grad(lambda t: (f(t) * dy).sum(dtype=FP))(x), *ref["dx"], "grad")
    y, tangent = torch.func.jvp(f, (x,), (x.flip(0),))
    check(y, *ref["y"], "jvp")
    check_tangent(tangent, x.flip(0), y, dy, ref["dx"])
    other = x.flip(0) + 1
    want = oracle(other, dy)["y"]
    check(make_fx(f)(x)(other), *want, "make_fx")
    check(torch.jit.trace(f, (x,), check_trace=False)(other), *want, "jit")
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        assert f(mode.from_tensor(x)).shape == dy.shape
    kernels.reset()
    check(f(x), *ref["y"], "kernel")
    assert not kernels.counts()["fallback"]
    check_status()


@pytest.mark.parametrize("name", ["rms", "layer", "dropout", "ffn"])
def test_incoming_gradients_that_no_kernel_can_take(name):
    """Several gradients at once, gradients with a tangent, and a recorded backward pass: x itself is an ordinary tensor,
    so the forward pass ran the kernels; the backward pass goes through the formulas."""
    import torch.autograd.forward_ad as fwad
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x, dy, oracle = _transform_cases()[name]
    leaf = x.clone().requires_grad_(True)
    y = f(leaf)

    def grad(d, **kw):
        return torch.autograd.grad(y, leaf, d, retain_graph=True, **kw)[0]
    many = torch.stack([dy, dy.flip(0), -2 * dy])
    got = grad(many, is_grads_batched=True)
    for i in range(3):
        check(got[i], *oracle(x, many[i])["dx"], i)
    with fwad.dual_level():  # the backward pass is linear in dy: its tangent is that of dy, sent through it
        dx, tangent = fwad.unpack_dual(grad(fwad.make_dual(dy, many[1])))
        check(dx, *oracle(x, dy)["dx"], "dual")
        check(tangent, *oracle(x, many[1])["dx"], "tangent")
    check(make_fx(grad)(dy)(many[2]), *oracle(x, many[2])["dx"], "make_fx")
    check(grad(dy), *oracle(x, dy)["dx"], "kernel")


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu"])
def test_gated_ffn_gradients_from_the_formulas(act):
    """All gradients of a backward pass that no kernel can take, with leading dimensions and a residual."""
    x, w13, w2, res, dy = ffn_inputs(24, 64, 40, 72, BF, seed=35)
    leaves = [t.clone().requires_grad_(True) for t in (x.view(2, 3, 4, 64), w13, w2, res.view(2, 3, 4, 72))]
    y = gated_ffn(*leaves[:3], act=act, residual=leaves[3])
    many = torch.stack([dy, dy.flip(0)])
    got = torch.autograd.grad(y, leaves, many.view(2, 2, 3, 4, 72), is_grads_batched=True)
    for i in range(2):
        ref = ffn_oracle(x, w13, w2, res, many[i], act)
        for k, t in zip(("dx", "dw13", "dw2"), got):
            check(t[i].reshape(ref[k][0].shape), *ref[k], (k, i))
    assert torch.equal(got[3].view_as(many), many)


def test_lazily_negated_views():
    def lazy(t):  # t's values in a view whose memory holds -t
        v = torch.complex(torch.zeros_like(t.float()), -t.float()).to(torch.complex32 if t.dtype == HF else torch.complex64)
        v = v.conj().imag
        assert v.is_neg() and torch.equal(v, t)
        return v
    x, w, b, dy = norm_inputs(9, 40, FP, FP, seed=32)
    for rms in (True, False):
        ref = norm_oracle(x, w, None if rms else b, dy, 1e-6, rms)
        for k in range(4):
            got = run_norm(*(lazy(t) if i == k else t for i, t in enumerate((x, w, b))), lazy(dy) if k == 3 else dy, 1e-6, rms)
            for n in got:
                check(got[n], *ref[n], (n, k))
    assert torch.equal(fused.dropout(lazy(x), 0.3, 2, residual=dy), fused.dropout(x, 0.3, 2, residual=dy))
    assert torch.equal(fused.dropout(x, 0.3, 2, residual=lazy(dy)), fused.dropout(x, 0.3, 2, residual=dy))
    leaf = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(fused.dropout(leaf, 0.3, 2), leaf, lazy(dy))[0], fused.dropout(dy, 0.3, 2))
    t = ffn_inputs(9, 64, 40, 72, HF, seed=33)
    ref = ffn_oracle(*t, "silu")
    for k in range(5):
        x, w13, w2, res, dy = (lazy(v) if i == k else v for i, v in enumerate(t))
        leaves = [v.detach().requires_grad_(True) for v in (x, w13, w2)]
        y = gated_ffn(*leaves, residual=res)
        for n, got in zip(("y", "dx", "dw13", "dw2"), (y.detach(), *torch.autograd.grad(y, leaves, dy))):
            check(got, *ref[n], (n, k))


@pytest.mark.parametrize("name", ["rms", "layer", "dropout", "ffn"])
def test_forward_mode_tangents(name):
    """In a sum with x, where a dropped tangent would leave that of x; and tangents of the weights alone."""
    import torch.autograd.forward_ad as fwad
    f, x, dy, oracle = _transform_cases()[name]
    ref, t = oracle(x, dy), x.flip(0)
    with fwad.dual_level():
        xd = fwad.make_dual(x, t)
        kernels.reset()
        y, tangent = fwad.unpack_dual(f(xd))
        check(y, *ref["y"], "y")
        check_tangent(tangent, t, y, dy, ref["dx"])
        if name != "ffn":
            total = fwad.unpack_dual(xd + f(xd)).tangent
            assert torch.equal(total, t + tangent)
        assert not any(kernels.counts()["native"].values())
        if name in ("rms", "layer"):
            w, b = norm_inputs(12, 264, FP, FP, seed=30)[1:3]
            wd = fwad.make_dual(w, w.flip(0))
            y = fused.rms_norm(x, wd, 1e-6) if name == "rms" else fused.layer_norm(x, wd, b, 1e-6)
            check_tangent(fwad.unpack_dual(y).tangent, w.flip(0), x, dy, ref["dw"])
        f(x)  # an open level without tangents changes nothing
        assert kernels.counts()["native"] or name == "ffn"


def test_registry_none_is_plain_torch_everywhere():
    """``none`` holds for the block as well, whose name is opt-in; any list leaves a call of the block itself native."""
    x, w13, w2, res, dy = ffn_inputs(20, 64, 40, 72, BF, seed=34)
    ref = ffn_oracle(x, w13, w2, res, dy, "silu")
    old = {n for n in kernels.NAMES if kernels.enabled(n)}
    try:
        for spec, native in (("none", 0), ("rms_norm", 1), ("all", 1), ("gated_ffn", 1)):
            kernels.enable(spec)
            kernels.reset()
            check(gated_ffn(x, w13, w2, residual=res), *ref["y"], spec)
            assert kernels.counts()["native"].get("gated_ffn", 0) == native
            with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
                gated_ffn(x, w13, w2)
                torch.cuda.synchronize()
            names = [e.key for e in prof.key_averages()]
            assert names and any("afb::ffn::" in n for n in names) == bool(native), names
    finally:
        kernels.enable(sorted(old))
