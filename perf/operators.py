"""Cases for the trainer's feed-forward operators: the gated feed-forward block, the norms with trainable weights and
counter-based dropout, each forward and (``train``) with its gradients.

``own`` False computes them from elementary torch operations in fp32, rounded once; ``own`` True calls this package.
"""
import functools
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token through the drafter's feed-forward (hidden 2048, intermediate 6144): the weights' bytes
        dict(name="ffn_one_token", op="ffn", rows=1, hidden=2048, inter=6144, act="silu", dtype="bf16", train=False,
             residual=False),
        # a verify window of 16 sessions x 5 positions through the 640-wide shared expert of the 2560-wide model
        dict(name="ffn_verify_window", op="ffn", rows=80, hidden=2560, inter=640, act="silu", dtype="bf16",
             train=False, residual=True),
        # a prompt scored by the drafter (evaluation, no gradients), ragged length
        dict(name="ffn_prompt", op="ffn", rows=1999, hidden=2048, inter=6144, act="silu", dtype="bf16", train=False,
             residual=False),
        # one packed 16k training bin through the 512-wide shared expert of the 2048-wide model
        dict(name="ffn_train_shared", op="ffn", rows=16384, hidden=2048, inter=512, act="silu", dtype="bf16",
             train=True, residual=False),
        # drafter training: 1,025 anchors x 4 slots through its feed-forward
        dict(name="ffn_train_drafter", op="ffn", rows=4100, hidden=2048, inter=6144, act="silu", dtype="bf16",
             train=True, residual=True),
        # fp16 with tanh-GELU at the vision tower's widths, odd row count
        dict(name="ffn_train_gelu_fp16", op="ffn", rows=1237, hidden=1152, inter=4304, act="gelu_tanh", dtype="fp16",
             train=True, residual=False),
        # a short fine-tuning sequence
        dict(name="norm_short", op="norm", kind="rms", rows=37, width=2048, dtype="bf16", wdtype="fp32", train=True),
        # the vision tower's block norm over one image's patches
        dict(name="norm_patches", op="norm", kind="layer", rows=5632, width=1152, dtype="bf16", wdtype="bf16",
             train=False),
        # the post-shuffle merger norm of four images, trained
        dict(name="norm_train_merger", op="norm", kind="layer", rows=5633, width=4608, dtype="bf16", wdtype="fp32",
             train=True),
        # the drafter's fp32 norms over a 16k context
        dict(name="norm_train_fp32", op="norm", kind="rms", rows=16383, width=2048, dtype="fp32", wdtype="fp32",
             train=True),
        # dropout on the input of a LoRA adapter over a packed 16k bin, both directions
        dict(name="dropout_lora_input", op="dropout", rows=16384, width=2560, p=0.05, dtype="bf16", train=True,
             residual=False),
        # residual dropout in fp32 with a row width that is no multiple of the vector
        dict(name="dropout_residual_odd", op="dropout", rows=2047, width=1001, p=0.1, dtype="fp32", train=True,
             residual=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "norm", "dropout"])
    train = rng.random() < 0.6
    if op == "ffn":
        hidden = 8 * _log_int(rng, 128, 320)
        inter = 8 * _log_int(rng, 16, 768)
        most = 4100 * 2048 * 6144 // (hidden * inter)
        rows = _log_int(rng, 1, max(1, min(16384, most)))
        return dict(op=op, rows=rows, hidden=hidden, inter=inter, act=rng.choice(["silu", "gelu_tanh", "gelu"]),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), train=train, residual=rng.random() < 0.5)
    if op == "norm":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        width = _log_int(rng, 128, 8192)
        return dict(op=op, kind=rng.choice(["layer", "rms"]), rows=_log_int(rng, 16, 16384), width=width, dtype=dtype,
                    wdtype=rng.choice([dtype, "fp32"]), train=train)
    return dict(op=op, rows=_log_int(rng, 16, 16384), width=_log_int(rng, 128, 2560), p=round(rng.uniform(0.01, 0.5), 3),
                dtype=rng.choice(["bf16", "fp16", "fp32"]), train=train, residual=rng.random() < 0.5)


# ----------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    dt = _DT[case["dtype"]]

    def rn(*shape, s=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * s).to(dtype)

    st = {"case": case}
    T = case["rows"]
    if case["op"] == "ffn":
        H, F = case["hidden"], case["inter"]
        st["x"] = rn(T, H)  # rows as a norm leaves them
        st["w13"] = rn(2 * F, H, s=1.0 / math.sqrt(H))
        st["w2"] = rn(H, F, s=1.0 / math.sqrt(F))
        st["residual"] = rn(T, H) if case["residual"] else None
        st["dy"] = rn(T, H) if case["train"] else None
    elif case["op"] == "norm":
        W = case["width"]
        scale = torch.exp(torch.randn(T, 1, generator=g, device="cuda"))  # rows of different sizes and offsets
        st["x"] = ((torch.randn(T, W, generator=g, device="cuda") + 0.5) * scale).to(dt)
        wd = _DT[case["wdtype"]]
        st["w"] = rn(W, s=0.2, dtype=wd) + (1 if case["kind"] == "layer" else 0)
        st["b"] = rn(W, s=0.2, dtype=wd) if case["kind"] == "layer" else None
        st["dy"] = rn(T, W) if case["train"] else None
    else:
        W = case["width"]
        st["x"] = rn(T, W)
        st["residual"] = rn(T, W) if case["residual"] else None
        st["dy"] = rn(T, W) if case["train"] else None
        ints = torch.randint(0, 2**62, (2,), generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFFFFFF))
        st["seed"], st["offset"] = int(ints[0]), int(ints[1]) >> 20
    if case["train"]:  # what is trained is a leaf that asks for its gradient
        for k in ("x", "w13", "w2", "w", "b"):
            if st.get(k) is not None:
                st[k].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------------- plain forms
def _act(name, g):
    """act(g) and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def _plain_ffn(st):
    case = st["case"]
    F, dt = case["inter"], st["x"].dtype
    x, w13, w2 = st["x"].float(), st["w13"].float(), st["w2"].float()
    gu = x @ w13.t()
    g, u = gu[:, :F], gu[:, F:]
    a, da = _act(case["act"], g)
    h = a * u
    y = h @ w2.t()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    if not case["train"]:
        return {"y": y.to(dt)}
    dy = st["dy"].float()
    dh = dy @ w2
    dgu = torch.cat([dh * u * da, dh * a], 1)
    return {"y": y.to(dt), "dx": (dgu @ w13).to(dt), "dw13": (dgu.t() @ x).to(dt), "dw2": (dy.t() @ h).to(dt)}


def _plain_norm(st):
    case = st["case"]
    x, w = st["x"].float(), st["w"].float()
    layer = case["kind"] == "layer"
    xc = x - x.mean(-1, keepdim=True) if layer else x
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + _EPS)
    xh = xc * rstd
    m = w if layer else 1 + w
    y = xh * m + (st["b"].float() if layer else 0)
    out = {"y": y.to(st["x"].dtype)}
    if case["train"]:
        dy = st["dy"].float()
        v = dy * m
        dx = v - xh * (v * xh).mean(-1, keepdim=True)
        if layer:
            dx = dx - v.mean(-1, keepdim=True)
            out["db"] = dy.sum(0).to(st["b"].dtype)
        out["dx"] = (dx * rstd).to(st["x"].dtype)
        out["dw"] = (dy * xh).sum(0).to(st["w"].dtype)
    return out


def _mulhilo(a, m):
    """High and low 32 bits of a * m, for a < 2^32 held in int64."""
    hi_part, lo_part = a * (m >> 16), a * (m & 0xFFFF)
    mid = hi_part + (lo_part >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (lo_part & 0xFFFF)


def _round(s, key):
    h0, l0 = _mulhilo(s[0], 0xD2511F53)
    h1, l1 = _mulhilo(s[2], 0xCD9E8D57)
    return h1 ^ s[1] ^ key[0], l1, h0 ^ s[3] ^ key[1], l0


def _keep(n, p, seed, offset, device):
    """Which of n elements stay: Philox4x32-10 with the 64-bit key `seed` and the counter offset + i // 8 gives 128
    bits for eight elements, 16 bits each, lowest first; an element stays where they are below the threshold."""
    t = int((1 - p) * 65536 + 0.5)
    c = torch.arange((n + 7) // 8, device=device) + offset
    keys = [((seed + 0) % 2**32, (seed >> 32) % 2**32)]
    keys = functools.reduce(lambda ks, _: ks + [((ks[-1][0] + 0x9E3779B9) % 2**32, (ks[-1][1] + 0xBB67AE85) % 2**32)],
                            range(9), keys)
    zero = torch.zeros_like(c)
    s = functools.reduce(_round, keys, (c & 0xFFFFFFFF, (c >> 32) & 0xFFFFFFFF, zero, zero))
    bits = torch.stack([s[0] & 0xFFFF, s[0] >> 16, s[1] & 0xFFFF, s[1] >> 16, s[2] & 0xFFFF, s[2] >> 16,
                        s[3] & 0xFFFF, s[3] >> 16], 1).reshape(-1)[:n]
    return bits < t, 65536 / t


def _plain_dropout(st):
    case, x = st["case"], st["x"]
    keep, scale = _keep(x.numel(), case["p"], st["seed"], st["offset"], x.device)
    keep = keep.view(x.shape)
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * scale, zero)
    if st["residual"] is not None:
        y = y + st["residual"].float()
    out = {"y": y.to(x.dtype)}
    if case["train"]:
        out["dx"] = torch.where(keep, st["dy"].float() * scale, zero).to(x.dtype)
    return out


# --------------------------------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"ffn": _plain_ffn, "norm": _plain_norm, "dropout": _plain_dropout}[case["op"]](state)
    from arc_forge_2026_b200.train import fused
    from arc_forge_2026_b200.train.ffn import gated_ffn
    x = state["x"]
    if case["op"] == "ffn":
        y = gated_ffn(x, state["w13"], state["w2"], act=case["act"], residual=state["residual"])
        asked = {"dx": x, "dw13": state["w13"], "dw2": state["w2"]}
    elif case["op"] == "norm":
        if case["kind"] == "layer":
            y = fused.layer_norm(x, state["w"], state["b"], _EPS)
            asked = {"db": state["b"], "dx": x, "dw": state["w"]}
        else:
            y = fused.rms_norm(x, state["w"], _EPS)
            asked = {"dx": x, "dw": state["w"]}
    else:
        y = fused.dropout(x, case["p"], state["seed"], state["offset"], residual=state["residual"])
        asked = {"dx": x}
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, list(asked.values()), state["dy"])
    return {"y": y.detach(), **dict(zip(asked, grads))}


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    T = case["rows"]
    if case["op"] == "ffn":
        H, F = case["hidden"], case["inter"]
        rows, weights = T * H * e, 3 * F * H * e
        fwd = 6 * T * H * F
        if not case["train"]:
            return {"bytes": rows * (2 + case["residual"]) + weights, "flops": fwd}
        return {"bytes": rows * (4 + case["residual"]) + 2 * weights, "flops": 3 * fwd}
    n = T * case["width"]
    if case["op"] == "norm":
        we = 4 if case["wdtype"] == "fp32" else 2
        vec = case["width"] * we * (2 if case["kind"] == "layer" else 1)
        if not case["train"]:
            return {"bytes": 2 * n * e + vec, "flops": 8 * n}
        return {"bytes": 4 * n * e + 2 * vec, "flops": 20 * n}
    return {"bytes": n * e * (2 + case["residual"] + 2 * case["train"]), "flops": n * (2 + case["train"])}


# ------------------------------------------------------------------------------------------------------------- exact
def _exact_keep(n, p, seed, offset):
    """The mask once more, in numpy's unsigned integers."""
    t = int(math.floor((1 - p) * 65536 + 0.5))
    m32 = np.uint64(0xFFFFFFFF)
    sh = np.uint64(32)
    ctr = np.arange((n + 7) // 8, dtype=np.uint64) + np.uint64(offset)
    x0, x1, x2, x3 = ctr & m32, ctr >> sh, np.zeros_like(ctr), np.zeros_like(ctr)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = (b >> sh) ^ x1 ^ np.uint64(k0), b & m32, (a >> sh) ^ x3 ^ np.uint64(k1), a & m32
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack([x0, x1, x2, x3], 1).astype("<u4")
    return words.view("<u2").reshape(-1)[:n] < t, 65536.0 / t


def exact(case, seed):
    st = {k: (v.detach().double() if isinstance(v, torch.Tensor) else v) for k, v in prepare(case, seed).items()}
    x = st["x"]
    if case["op"] == "ffn":
        Fi = case["inter"]
        gate, up = x @ st["w13"][:Fi].T, x @ st["w13"][Fi:].T
        gate.requires_grad_(True)
        if case["act"] == "silu":
            f = torch.nn.functional.silu(gate)
        else:
            f = torch.nn.functional.gelu(gate, approximate="tanh" if case["act"] == "gelu_tanh" else "none")
        hid = f.detach() * up
        y = hid @ st["w2"].T + (st["residual"] if case["residual"] else 0)
        if not case["train"]:
            return {"y": y}
        back = st["dy"] @ st["w2"]
        (dgate,) = torch.autograd.grad(f, gate, back * up)
        dup = back * f.detach()
        return {"y": y, "dx": dgate @ st["w13"][:Fi] + dup @ st["w13"][Fi:],
                "dw13": torch.cat([dgate.T @ x, dup.T @ x]), "dw2": st["dy"].T @ hid}
    if case["op"] == "norm":
        x.requires_grad_(True)
        w = st["w"].requires_grad_(True)
        if case["kind"] == "layer":
            b = st["b"].requires_grad_(True)
            y = torch.nn.functional.layer_norm(x, (case["width"],), w, b, _EPS)
            names, leaves = ("db", "dx", "dw"), (b, x, w)
        else:
            y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * (1 + w)
            names, leaves = ("dx", "dw"), (x, w)
        if not case["train"]:
            return {"y": y.detach()}
        return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, st["dy"])))}
    keep, scale = _exact_keep(x.numel(), case["p"], st["seed"], st["offset"])
    keep = torch.from_numpy(keep).to(x.device).view(x.shape).double()
    y = x * keep * scale
    if case["residual"]:
        y = y + st["residual"]
    return {"y": y, "dx": st["dy"] * keep * scale} if case["train"] else {"y": y}
