"""Fused training ops of the QAD student (``csrc/train_fused.cu``): one kernel each way instead of a chain of
PyTorch element-wise ops, bf16 in and out with fp32 math, fixed-order reductions.

Each function takes the student's tensors as they are (strided views included) and falls back to the plain-torch
math of ``models.reference`` off the GPU, or when a shape is outside what the kernels cover; the CPU paths are the
oracles the GPU tests compare against. The reference's counterparts are its fused Triton training kernels
(``training/work/qwen38fn_lora/trainer_kernels.py:234-290`` GatedRMSNormFLA, ``int3_moe.py:108-152,376-430``
SwiGLU and token aggregation, ``fp8_moe.py`` _swiglu_backward / _routing_backward).

Beside them, with trainable weights: :func:`layer_norm` and :func:`rms_norm` (``csrc/norm_train.cu``) and
:func:`dropout` from a counter-based generator (``csrc/dropout.cu``); the gated feed-forward block is ``train/ffn.py``.
These four take their plain forms inside function transforms (``torch.func``), in forward-mode differentiation, under
dispatch modes, while a trace is recorded, and for tensors whose memory is not their value (fake tensors, other
subclasses, lazily negated views).
"""
from __future__ import annotations

import functools

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ..models import reference as R
from . import kernels

_BF = torch.bfloat16
_NORM_H = (128, 256, 512, 1024, 2048)


@functools.cache
def _ext():
    from ..ops import C
    return C()


def _gpu_bf16(*ts) -> bool:  # (tensors that dispatch to Python, fake ones among them, have no memory to read)
    return all(t.is_cuda and t.dtype == _BF and t.stride(-1) == 1
               and type(t).__torch_dispatch__ is torch.Tensor.__torch_dispatch__ for t in ts)


class _ConvSiLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, pos):
        y = torch.empty(x.shape, dtype=_BF, device=x.device)
        _ext().conv_silu(x, w, y, None, None, pos)
        ctx.save_for_backward(x, w, pos)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, pos = ctx.saved_tensors
        dx = torch.empty(x.shape, dtype=_BF, device=x.device)
        _ext().conv_silu(x, w, dx, dy.to(_BF).contiguous(), dx, pos)
        return dx, None, None


def conv_silu(x: torch.Tensor, w: torch.Tensor, pos: torch.Tensor | None = None) -> torch.Tensor:
    """Causal depthwise conv (kernel 4, zero history) + SiLU over x [B, T, C] (a strided view is fine); frozen w.
    ``pos`` [B, T] (packed sequences): each token's position inside its sequence; taps before the start read 0."""
    if (kernels.use("conv_silu") and _gpu_bf16(x) and x.dim() == 3 and w.shape[-1] == 4 and x.shape[-1] % 8 == 0
            and x.stride(1) % 8 == 0 and x.stride(0) == x.shape[1] * x.stride(1) and not w.requires_grad):
        kernels.hit("conv_silu", True)
        return _ConvSiLU.apply(x, w.float().contiguous(), None if pos is None else pos.int().contiguous())
    if x.is_cuda:
        kernels.hit("conv_silu", False)
    if pos is None:
        return R.causal_conv1d(x, w)[0]
    return conv_silu_reference(x, w, pos)


def conv_silu_reference(x, w, pos):
    """Plain-torch causal conv + SiLU with per-token sequence positions (the packed-sequence oracle)."""
    B, T, Cc = x.shape
    K = w.shape[1]
    xf = x.float()
    pre = torch.zeros(B, T, Cc, dtype=torch.float32, device=x.device)
    for k in range(K):
        lag = K - 1 - k
        if lag >= T:
            continue
        shifted = torch.zeros_like(xf)
        shifted[:, lag:] = xf[:, : T - lag]
        live = (pos >= lag).to(xf.dtype)[..., None]
        pre = pre + w[:, k].float() * shifted * live
    return F.silu(pre).to(x.dtype)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps, z):
        H = x.shape[-1]
        y = torch.empty(x.shape, dtype=_BF, device=x.device)
        rstd = torch.empty(x.numel() // H, dtype=torch.float32, device=x.device)
        _ext().rmsnorm_train(x, z, w, eps, y, rstd, None, None, None)
        ctx.save_for_backward(x, w, rstd, z)
        ctx.eps = eps
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, rstd, z = ctx.saved_tensors
        dx = torch.empty(x.shape, dtype=_BF, device=x.device)
        dz = torch.empty(z.shape, dtype=_BF, device=x.device) if z is not None else None
        _ext().rmsnorm_train(x, z, w, ctx.eps, dx, rstd, dy.to(_BF).contiguous(), dx, dz)
        return dx, None, None, dz


def _norm_ok(x, w) -> bool:
    return _gpu_bf16(x) and x.shape[-1] in _NORM_H and x.dim() >= 2 and not w.requires_grad


_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_NORM_MAX_WIDTH = 16384


def _train_norm_ok(x, w) -> bool:
    return (x.is_cuda and w.device == x.device and x.dtype in _FLOATS and w.dtype in (x.dtype, torch.float32)
            and 1 <= x.shape[-1] <= _NORM_MAX_WIDTH)


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """Zero-centred RMSNorm ``x / rms(x) * (1 + w)`` of ``models.reference.rms_norm``: a frozen w at the model's widths
    in bf16 on the student's kernel, a trainable w (gradient of w in w's type), any other width up to 16,384, fp16
    and fp32 on the trainable norm's."""
    if kernels.use("rms_norm") and not w.requires_grad and _norm_ok(x, w):
        kernels.hit("rms_norm", True)
        return _RMSNorm.apply(x, w.float().contiguous(), eps, None)
    if kernels.use("rms_norm") and w.shape == x.shape[-1:] and _train_norm_ok(x, w):
        y = _ext().train_norm(x, w, None, eps, True)
        if y is not None:
            kernels.hit("rms_norm", True)
            return y
    if x.is_cuda:
        kernels.hit("rms_norm", False)
    return R.rms_norm(x, w, eps)


def layer_norm_reference(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None, eps: float) -> torch.Tensor:
    """LayerNorm over the last dim in fp32 (fp64 for fp64 inputs), rounded once to x's type."""
    ct = torch.promote_types(x.dtype, torch.float32)
    z = x.to(ct)
    z = z - z.mean(-1, keepdim=True)
    y = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + eps) * w.to(ct)
    return (y if b is None else y + b.to(ct)).to(x.dtype)


def layer_norm(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm ``(x - mean) / sqrt(var + eps) * w (+ b)`` over the last dim (1 to 16,384 wide), differentiable in x, w
    and b; x bf16, fp16 or fp32, w and b in x's type or fp32 (their gradients come in their own type).
    Statistics and sums are fp32 and of fixed order."""
    if x.dim() < 1 or w.shape != x.shape[-1:] or (b is not None and b.shape != w.shape):
        raise ValueError(f"layer_norm: x {tuple(x.shape)}, w {tuple(w.shape)}"
                         + ("" if b is None else f", b {tuple(b.shape)}"))
    if w.device != x.device or (b is not None and (b.device != w.device or b.dtype != w.dtype)):
        raise ValueError("layer_norm: w and b on x's device, b in w's type")
    if kernels.use("layer_norm") and _train_norm_ok(x, w):
        y = _ext().train_norm(x, w, b, eps, False)
        if y is not None:
            kernels.hit("layer_norm", True)
            return y
    if x.is_cuda:
        kernels.hit("layer_norm", False)
    return layer_norm_reference(x, w, b, eps)


def _i64(v: int) -> int:
    """v mod 2^64 as a signed 64-bit integer."""
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v


def dropout_threshold(p: float) -> int:
    """An element stays when its 16 random bits are below this: (1 - p) in 2^-16 steps."""
    return int((1.0 - p) * 65536 + 0.5)


def dropout_keep_reference(n: int, p: float, seed: int, offset: int = 0, device=None) -> torch.Tensor:
    """Which of n elements :func:`dropout` keeps: element i takes bits 16 (i % 8) .. of the 128-bit output of
    Philox4x32-10 with key ``seed`` and counter ``offset + i // 8``."""
    m32 = 0xFFFFFFFF
    ctr = torch.arange((n + 7) // 8, dtype=torch.int64, device=device) + _i64(offset)
    s = [ctr & m32, (ctr >> 32) & m32, torch.zeros_like(ctr), torch.zeros_like(ctr)]
    k0, k1 = seed & m32, (seed >> 32) & m32

    def mul(a, m):  # 32 x 32 -> (high, low) without leaving int64
        lo = a * (m & 0xFFFF)
        mid = a * (m >> 16) + (lo >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)
    for _ in range(10):
        ah, al = mul(s[0], 0xD2511F53)
        bh, bl = mul(s[2], 0xCD9E8D57)
        s = [bh ^ s[1] ^ k0, bl, ah ^ s[3] ^ k1, al]
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    bits = torch.stack([(v >> sh) & 0xFFFF for v in s for sh in (0, 16)], 1).reshape(-1)[:n]
    return bits < dropout_threshold(p)


def _dropout_plain(x, residual, p, seed, offset, rng):
    if rng is not None:
        seed, offset = seed + int(rng[0]), offset + int(rng[1])
    keep = dropout_keep_reference(x.numel(), p, seed, offset, x.device).view(x.shape)
    t = dropout_threshold(p)
    ct = torch.promote_types(x.dtype, torch.float32)
    y = torch.where(keep, x.to(ct) * (65536.0 / t if t else 0.0), torch.zeros((), dtype=ct, device=x.device))
    return (y if residual is None else y + residual.to(ct)).to(x.dtype)


class _DropoutPlain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, rng):
        ctx.save_for_backward(rng)
        ctx.args = (p, seed, offset)
        return _dropout_plain(x, residual, p, seed, offset, rng)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = _dropout_plain(dy, None, *ctx.args, *ctx.saved_tensors) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x: torch.Tensor, p: float, seed, offset: int = 0, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``x`` with elements dropped with probability ``p`` and the rest scaled by 1 / (1 - p), plus ``residual`` if given
    (``csrc/dropout.cu``). The mask is a pure function of (seed, offset) and the element's index in x's row-major
    order; it is never stored, the backward pass makes it again, and CPU and GPU agree on it. A call uses the counters
    ``offset .. offset + ceil(numel / 8) - 1`` of ``seed``: calls whose ranges do not meet are independent.

    p in [0, 1] is taken in steps of 2^-16 (the scale is that of the rounded p, so the expectation is exact); a dropped
    element is 0 whatever it held. ``seed``: an int, or an int64 tensor [2] = (seed, offset) on x's device, read when
    the kernel runs (a captured graph draws anew when the tensor is updated between replays; not between a forward and
    its backward); ``offset`` is added to the tensor's."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p = {p} is not in [0, 1]")
    rng = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.shape != (2,) or seed.device != x.device:
            raise ValueError("dropout: the seed tensor is int64 [2] (seed, offset) on x's device")
        rng, seed = seed.contiguous(), 0
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError("dropout: residual has x's shape, type and device")
    if not x.is_floating_point():
        raise ValueError(f"dropout: x is {x.dtype}")
    if x.is_cuda and x.dtype in _FLOATS and kernels.use("dropout"):
        y = _ext().dropout(x, residual, dropout_threshold(p), _i64(int(seed)), _i64(int(offset)), rng)
        kernels.hit("dropout", y is not None)
        # what the kernel cannot read goes through operations that can be transformed and traced
        return _dropout_plain(x, residual, float(p), int(seed), int(offset), rng) if y is None else y
    if x.is_cuda:
        kernels.hit("dropout", False)
    return _DropoutPlain.apply(x, residual, float(p), int(seed), int(offset), rng)


def gated_rms_norm(x: torch.Tensor, z: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    """GDN output norm ``x / rms(x) * w * silu(z)`` (frozen w) of ``models.reference.gated_rms_norm``."""
    if kernels.use("gated_rms_norm") and _norm_ok(x, w) and _gpu_bf16(z) and z.shape == x.shape:
        kernels.hit("gated_rms_norm", True)
        return _RMSNorm.apply(x, w.float().contiguous(), eps, z)
    if x.is_cuda:
        kernels.hit("gated_rms_norm", False)
    return R.gated_rms_norm(x, z, w, eps)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        I = gu.shape[-1] // 2
        h = torch.empty(*gu.shape[:-1], I, dtype=_BF, device=gu.device)
        _ext().swiglu_train(gu, h, None)
        ctx.save_for_backward(gu)
        return h

    @staticmethod
    def backward(ctx, dh):
        (gu,) = ctx.saved_tensors
        dgu = torch.empty_like(gu)
        _ext().swiglu_train(gu, dgu, dh.to(_BF).contiguous())
        return dgu


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` of ``gu = [gate | up]`` along the last dim."""
    I = gu.shape[-1] // 2
    if kernels.use("swiglu") and _gpu_bf16(gu) and gu.is_contiguous() and I % 8 == 0:
        kernels.hit("swiglu", True)
        return _SwiGLU.apply(gu)
    if gu.is_cuda:
        kernels.hit("swiglu", False)
    return F.silu(gu[..., :I].float()).to(gu.dtype) * gu[..., I:]


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, inv, w):
        out = torch.empty(w.shape[0], y.shape[1], dtype=_BF, device=y.device)
        _ext().moe_combine_train(y, inv, w, out, None, None, None)
        ctx.save_for_backward(y, inv, w)
        return out

    @staticmethod
    def backward(ctx, dout):
        y, inv, w = ctx.saved_tensors
        dy, dw = torch.empty_like(y), torch.empty_like(w)
        _ext().moe_combine_train(y, inv, w, dy, dout.to(_BF).contiguous(), dy, dw)
        return dy, None, dw


def moe_combine(y: torch.Tensor, inv: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """out[t] = sum_k w[t, k] y[inv[t*K + k]]: routed rows (expert order) back to their tokens, weighted."""
    T, K = w.shape
    H = y.shape[-1]
    if kernels.use("moe_combine") and _gpu_bf16(y) and y.is_contiguous() and H in (256, 512, 1024, 2048):
        kernels.hit("moe_combine", True)
        return _Combine.apply(y, inv.contiguous(), w.float().contiguous())
    if y.is_cuda:
        kernels.hit("moe_combine", False)
    yt = y.index_select(0, inv).view(T, K, H)
    return (yt * w.to(yt.dtype)[..., None]).sum(1)


class _Dispatch(torch.autograd.Function):
    """xs = x[order // K] (every token once per routed expert, in expert order); the gradient sums each token's K
    rows through the inverse permutation in one kernel."""

    @staticmethod
    def forward(ctx, x, order, inv, K):
        ctx.save_for_backward(inv)
        ctx.K, ctx.T = K, x.shape[0]
        return x.index_select(0, torch.div(order, K, rounding_mode="floor"))

    @staticmethod
    def backward(ctx, g):
        (inv,) = ctx.saved_tensors
        g = g.to(_BF).contiguous()
        dx = torch.empty(ctx.T, g.shape[-1], dtype=_BF, device=g.device)
        _ext().moe_dispatch_bwd(g, inv, ctx.K, dx)
        return dx, None, None, None


def moe_dispatch(x: torch.Tensor, order: torch.Tensor, inv: torch.Tensor, K: int) -> torch.Tensor:
    if kernels.use("moe_dispatch") and _gpu_bf16(x) and x.shape[-1] in (256, 512, 1024, 2048):
        kernels.hit("moe_dispatch", True)
        return _Dispatch.apply(x, order, inv.contiguous(), K)
    if x.is_cuda:
        kernels.hit("moe_dispatch", False)
    return None
