"""Layer norm with trained weight and bias (csrc/layer_norm.cu).

``layer_norm(x, weight, bias, eps)`` normalises the last dimension of ``x``
(fp32 statistics, one rounding of the result) and is differentiable in all
three; ``layer_norm_forward`` / ``layer_norm_backward`` are its two halves for
callers that run their backward by hand.

``x`` is bf16, fp16 or fp32 of any leading shape; weight and bias have its type
or are fp32 (their gradients have the type of each).  ``bias`` may be None.
Statistics are fp32, the column sums of the backward too, added in an order
that does not depend on timing.  On the CPU the same functions compute with
PyTorch operations.

The reference keeps the vision tower's layer norms frozen
(src/graspo/backends/graspoflow/models/qwen3/model.py:170-232).
"""

from __future__ import annotations

import torch

from graspo_b200.ops._ext import ext, launches

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None) -> None:
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm needs a last dimension to normalise: {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise ValueError(f"layer_norm takes bf16, fp16 or fp32, not {x.dtype}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None and name == "bias":
            continue
        if p.shape != x.shape[-1:] or p.device != x.device or p.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be [{x.shape[-1]}] of x's type or fp32 on its device")


def _rows(t: torch.Tensor) -> torch.Tensor:
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
                       eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)``; the statistics are fp32, one per row."""
    _check(x, weight, bias)
    rows = _rows(x)
    if not x.is_cuda:
        f = rows.float()
        mean = f.mean(-1)
        c = f - mean[:, None]
        rstd = torch.rsqrt(c.square().mean(-1) + eps)
        y = c * rstd[:, None] * weight.float() + (0 if bias is None else bias.float())
        return y.to(x.dtype).view(x.shape), mean, rstd
    y = torch.empty(rows.shape, device=x.device, dtype=x.dtype)
    mean, rstd = torch.empty(2, rows.shape[0], device=x.device, dtype=torch.float32)
    ext().layer_norm_fwd(rows, weight.contiguous(), None if bias is None else bias.contiguous(), y, mean, rstd,
                         float(eps))
    return y.view(x.shape), mean, rstd


def layer_norm_backward(
    dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
    bias_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, dweight, dbias)`` from the forward's input and statistics; ``dbias``
    has ``bias_dtype`` (the weight's type when None)."""
    _check(x, weight, None)
    bias_dtype = bias_dtype or weight.dtype
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError(f"dy must be like x: {tuple(dy.shape)} {dy.dtype}, {tuple(x.shape)} {x.dtype}")
    if bias_dtype not in (x.dtype, torch.float32):
        raise ValueError("the bias has x's type or fp32")
    rows, g = _rows(x), _rows(dy)
    if mean.shape != (rows.shape[0],) or rstd.shape != mean.shape:
        raise ValueError("mean and rstd must hold one value per row of x")
    if not x.is_cuda:
        n = (rows.float() - mean[:, None]) * rstd[:, None]
        gf = g.float()
        a = gf * weight.float()
        dx = rstd[:, None] * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
        return dx.to(x.dtype).view(x.shape), (gf * n).sum(0).to(weight.dtype), gf.sum(0).to(bias_dtype)
    dx = torch.empty(rows.shape, device=x.device, dtype=x.dtype)
    dw = torch.empty(x.shape[-1], device=x.device, dtype=weight.dtype)
    db = torch.empty(x.shape[-1], device=x.device, dtype=bias_dtype)
    launches.add(1)                               # the join of the column sums
    ext().layer_norm_bwd(g, rows, weight.contiguous(), mean, rstd, dx, dw, db)
    return dx.view(x.shape), dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy, x, weight, mean, rstd, ctx.bias_dtype)
        return dx, dw, None if ctx.bias_dtype is None else db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) * rstd * weight + bias`` over the last dimension, differentiable in all three."""
    _check(x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, float(eps))
