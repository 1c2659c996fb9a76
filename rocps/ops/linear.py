"""Linear layer with its epilogue: ``y = act(x W^T + b) + r`` in one kernel.

The product runs on the matrix cores with fp32 sums; bias, activation and
residual are applied to the sums before they are rounded once to the type of
``x``.  Any number of rows and features, bfloat16 or float16
(csrc/kernels/linear_fwd.h, linear_rows.hip, linear_bwd.hip on the product of
tile_gemm.h); on the CPU the same in plain PyTorch, in float32 (float64 for
float64 inputs).  On the GPU a row has at most 2**22 - 8 values, x less than
2**30 rows and, in training, the weight 2**22 - 8 rows at most; more are
refused.

The backward pass keeps ``x`` and, where there is an activation, the
pre-activations ``p = x W^T + b`` in the type of ``x``, and computes

    g  = dy * act'(p)              rounded to that type for the products,
                                   in float16 to infinity past 65504
    dx = g W      dW = g^T x      db = sum over rows of g      dr = dy

db from the unrounded g.  (The gated layer keeps its two projections in 24
bits: g is a product of both, and their rounding to 16 would add as much error
as that of g itself.)  With ``checkpoint="8bit"`` it keeps x and p in 8 bits
(rocps/ops/act8.py), half the memory or less: dW and g are then those of the
kept values.  y is the same but for the order of its sums, which goes by sizes
and by what is kept.

A training step can be captured into a graph.  As for every layer, torch ties
a leaf's gradient to the stream of the autograd graph that is alive: drop the
outputs of eager steps on the same weights before the capture.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from rocps.ops import hip_ext, require_hip_for
from rocps.ops.act8 import pack_rows, unpack_rows

__all__ = ["linear_act"]

_ACTS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}
_C = 0.7978845608028654  # sqrt(2 / pi)
_A = 0.044715


def act_cpu(v: torch.Tensor, act: int) -> torch.Tensor:
    if act == 1:
        return v.clamp(min=0)
    if act == 2:
        return 0.5 * v * (1 + torch.tanh(_C * (v + _A * v ** 3)))
    if act == 3:
        return v * torch.sigmoid(v)
    return v


def slope_cpu(v: torch.Tensor, act: int) -> torch.Tensor:
    if act == 1:
        return (v > 0).to(v.dtype)
    if act == 2:  # 0 or 1 past 12, where v ** 2 may overflow
        v = v.clamp(-12, 12)
        t = torch.tanh(_C * (v + _A * v ** 3))
        return (0.5 * (1 + t)
                + 0.5 * v * (1 - t * t) * _C * (1 + 3 * _A * v ** 2))
    if act == 3:  # 0 or 1 at the infinities that a 16-bit type may hold
        most = torch.finfo(v.dtype).max
        v = v.clamp(-most, most)
        z = torch.sigmoid(v)
        return z * (1 + v * (1 - z))
    return torch.ones_like(v)


def wide(t: torch.Tensor) -> torch.Tensor:
    """In the type that the CPU computes in."""
    return t if t.dtype == torch.float64 else t.float()


def _check_cpu(op: str, x, weight, bias, checkpoint) -> None:
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{op}: x {tuple(x.shape)} and weight "
                         f"{tuple(weight.shape)} do not fit")
    if 0 in weight.shape:
        raise ValueError(f"{op}: weight {tuple(weight.shape)} is empty")
    if not x.is_floating_point():
        raise TypeError(f"{op}: {x.dtype} is no floating type")
    if checkpoint and x.dtype == torch.float64:
        raise TypeError(f"{op}: no 8-bit checkpoint of float64")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise TypeError(f"{op}: {name} is {t.dtype} on {t.device}, x is "
                            f"{x.dtype} on {x.device}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"{op}: bias {tuple(bias.shape)}, not "
                         f"({weight.shape[0]},)")


def forward_cpu(x, w, b, r, act: int, gated: bool, keep: int):
    pre = wide(x) @ wide(w).t()
    if b is not None:
        pre = pre + wide(b)
    if gated:
        half = pre.shape[1] // 2
        y = act_cpu(pre[:, :half], act) * pre[:, half:]
    else:
        y = act_cpu(pre, act)
    if r is not None:
        y = y + wide(r)
    if keep == 0 or act == 0:
        return y.to(x.dtype), None, None
    if keep == 1:  # the gated layer's in more than 16 bits, see the module
        return y.to(x.dtype), pre if gated else pre.to(x.dtype), None
    if gated:  # each half in groups of its own
        half = pre.shape[1] // 2
        (g, gs), (u, us) = pack_rows(pre[:, :half]), pack_rows(pre[:, half:])
        return (y.to(x.dtype), torch.cat([g, u], 1), torch.cat([gs, us], 1))
    return (y.to(x.dtype), *pack_rows(pre))


def backward_cpu(dy, x, x_scales, w, pre, scales, act: int, gated: bool,
                 k: int, need_x: bool, need_w: bool, need_b: bool):
    n = dy.shape[1]
    d = wide(dy)
    g = d
    if act != 0:
        if scales is None:
            pre = wide(pre)
        elif gated:
            c, s = pre.shape[1] // 2, scales.shape[1] // 2
            pre = torch.cat(
                [unpack_rows(pre[:, a * c:(a + 1) * c].contiguous(),
                             scales[:, a * s:(a + 1) * s].contiguous(),
                             dy.shape,
                             torch.float32) for a in (0, 1)], 1)
        else:
            pre = unpack_rows(pre, scales, dy.shape, torch.float32)
        if gated:
            a, u = pre[:, :n], pre[:, n:]
            g = torch.cat([d * u * slope_cpu(a, act), d * act_cpu(a, act)], 1)
        else:
            g = d * slope_cpu(pre, act)
    dx = dw = db = None
    if need_x:
        dx = (g @ wide(w)).to(dy.dtype)
    if need_w:
        if x_scales is not None:
            x = unpack_rows(x, x_scales, torch.Size((dy.shape[0], k)),
                            dy.dtype)
        dw = (g.t() @ wide(x)).to(dy.dtype)
    if need_b:
        db = g.sum(0).to(dy.dtype)
    return dx, dw, db


class _LayerFn(torch.autograd.Function):
    """Both layers on the CPU (the GPU's is in csrc/kernels/linear_ext.cc)."""

    @staticmethod
    def forward(ctx, x, w, b, r, act, gated, eight):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        need = need_x or need_w or need_b
        y, pre, scales = forward_cpu(x, w, b, r, act, gated,
                                     (2 if eight else 1) if need else 0)
        kept = x_scales = None
        if need_w:
            kept, x_scales = pack_rows(x) if eight else (x, None)
        ctx.save_for_backward(kept, x_scales, w if need_x else None, pre,
                              scales)
        ctx.act, ctx.gated, ctx.k = act, gated, x.shape[1]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = backward_cpu(dy, *ctx.saved_tensors, ctx.act,
                                      ctx.gated, ctx.k, *need[:3])
        return dx, dw, db, dy if need[3] else None, None, None, None


def layer(op: str, acts: dict, x, weight, bias, residual, activation,
          checkpoint, gated: bool) -> torch.Tensor:
    """What linear_act and gated_linear share."""
    try:
        act = acts[activation]
        eight = {None: False, "8bit": True}[checkpoint]
    except (KeyError, TypeError):
        raise ValueError(
            f"{op}: activation {activation!r}, checkpoint {checkpoint!r}: not "
            f"of {list(acts)} and [None, '8bit']") from None
    if require_hip_for(x):
        return hip_ext().linear_layer(x, weight, bias, residual, act, gated,
                                      eight)
    _check_cpu(op, x, weight, bias, eight)
    if gated and weight.shape[0] % 2:
        raise ValueError(f"{op}: weight {tuple(weight.shape)} has no two "
                         "halves")
    n = weight.shape[0] // 2 if gated else weight.shape[0]
    shape = x.shape[:-1] + (n,)
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"{op}: residual {tuple(residual.shape)}, not "
                             f"{tuple(shape)}")
        if residual.dtype != x.dtype or residual.device != x.device:
            raise TypeError(f"{op}: residual is {residual.dtype} on "
                            f"{residual.device}, x is {x.dtype} on {x.device}")
        residual = residual.reshape(shape[:-1].numel(), n)
    x = x.reshape(x.shape[:-1].numel(), x.shape[-1])
    return _LayerFn.apply(x, weight, bias, residual, act, gated,
                          eight).reshape(shape)


def linear_act(x: torch.Tensor, weight: torch.Tensor,
               bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, *,
               activation: Optional[str] = None,
               checkpoint: Optional[str] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    x (..., K), weight (N, K), bias (N,), residual (..., N) -> (..., N), all
    of one type on one device; ``activation`` None, "relu", "gelu" (tanh form)
    or "silu"; ``checkpoint`` None or "8bit" (see the module).  Rows may have
    any stride; whole multiples of 8 features from 16-byte aligned rows are
    used where they lie, others are copied first.  Differentiable once,
    backward; inputs with forward-mode tangents are refused."""
    return layer("linear_act", _ACTS, x, weight, bias, residual, activation,
                 checkpoint, False)
