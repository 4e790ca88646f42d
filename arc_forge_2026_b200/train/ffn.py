"""Gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) W2^T (+ residual)`` with its gradients
(``csrc/ffn.cu``): both input projections, the activation and the product are one tcgen05 kernel, the activation's
gradient is the epilogue of the down projection's backward product, and every product reads its operands where they
lie (no transposed copies).

    y = gated_ffn(x, w13, w2)                         # x [..., H], w13 = [Wg; Wu] [2F, H], w2 [N, F]
    y = gated_ffn(x, w13, w2, act="gelu_tanh", residual=r)

Types: bf16 or fp16, weights in x's type. Sums are fp32; ``h`` and the gradients of the two pre-activations are
rounded once to x's type (they are tensor-core operands); what the backward pass needs of the pre-activations is kept
in fp32 (8 F bytes a row; nothing when neither x nor w13 asks for a gradient). With few rows the forward pass keeps h
in two terms, so that only the result is rounded (dw2 is made from the first of them). In fp16 the rounded values have
fp16's range: an h, dg or du past 65,504 becomes infinite, and with it its row of y or dx and the weight gradients, where
the plain form, which rounds nothing before its result, may still be finite. Results do not depend on timing or on other work on the GPU: every
sum has a fixed order.

Off the GPU, in fp32, or when H, F or N is no multiple of 8 the plain-torch form runs, and so it does everywhere when
the kernel registry is ``none``. The student's shared experts and the drafter trainer's feed-forward use the block when
the registry name ``gated_ffn`` is enabled (``--fast-kernels all`` leaves it off, so their results stay what they were);
a call of :func:`gated_ffn` itself needs no name.
"""
from __future__ import annotations

import functools

import torch
import torch.nn.functional as F

from . import kernels

ACTS = {"silu": 0, "gelu_tanh": 1, "gelu": 2}


@functools.cache
def _ext():
    from ..ops import C
    return C()


def gated_ffn_reference(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, act: str = "silu",
                        residual: torch.Tensor | None = None) -> torch.Tensor:
    """The block in plain torch, in fp32 (fp64 for fp64 inputs), rounded once to x's type."""
    ct = torch.promote_types(x.dtype, torch.float32)
    I = w2.shape[1]
    gu = x.to(ct) @ w13.to(ct).t()
    g, u = gu[..., :I], gu[..., I:]
    a = F.silu(g) if act == "silu" else F.gelu(g, approximate="tanh" if act == "gelu_tanh" else "none")
    y = (a * u) @ w2.to(ct).t()
    if residual is not None:
        y = y + residual.to(ct)
    return y.to(x.dtype)


def _check(x, w13, w2, residual):
    if w13.dim() != 2 or w2.dim() != 2 or x.dim() < 1 or w13.shape[1] != x.shape[-1] \
            or w13.shape[0] != 2 * w2.shape[1]:
        raise ValueError(f"gated_ffn: x [..., H], w13 [2F, H], w2 [N, F]; got {tuple(x.shape)}, {tuple(w13.shape)}, "
                         f"{tuple(w2.shape)}")
    if 0 in (x.shape[-1], *w2.shape):
        raise ValueError("gated_ffn: empty feature dimension")
    for name, t in (("w13", w13), ("w2", w2), ("residual", residual)):
        if t is not None and (t.device != x.device or t.dtype != x.dtype):
            raise ValueError(f"gated_ffn: {name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    if residual is not None and residual.shape != (*x.shape[:-1], w2.shape[0]):
        raise ValueError(f"gated_ffn: residual {tuple(residual.shape)} does not fit x and w2")


def gated_ffn(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, act: str = "silu",
              residual: torch.Tensor | None = None) -> torch.Tensor:
    """``(act(g) * u) @ w2.T (+ residual)`` with ``[g | u] = x @ w13.T``; x [..., H], w13 [2F, H] (gate rows, then up
    rows), w2 [N, F], residual [..., N]; ``act``: ``silu``, ``gelu_tanh`` or ``gelu``. Differentiable (once) in x,
    w13, w2 and residual."""
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f"gated_ffn: unknown act {act!r}; known: {', '.join(ACTS)}")
    if x.is_cuda and kernels.any_enabled():
        # the binding checks the arguments and returns None for what the kernels do not cover
        y = _ext().gated_ffn(x, w13, w2, residual, code)
        kernels.hit("gated_ffn", y is not None)
        if y is not None:
            return y
    _check(x, w13, w2, residual)
    return gated_ffn_reference(x, w13, w2, act, residual)
