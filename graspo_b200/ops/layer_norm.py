"""Layer norm with trained weight and bias (csrc/layer_norm.cu).

``layer_norm(x, weight, bias, eps)`` normalises the last dimension of ``x``
(fp32 statistics, one rounding of the result) and is differentiable in all
three (once: a second derivative raises); ``layer_norm_forward`` /
``layer_norm_backward`` are its two halves for callers that run their backward by
hand.

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

from graspo_b200.ops._ext import err_word, ext, launches
from graspo_b200.ops._second import refuse_second

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None) -> None:
    """The kernels' own checks, for tensors that do not reach them."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm needs a last dimension to normalise: {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise ValueError(f"layer_norm takes bf16, fp16 or fp32, not {x.dtype}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None and name == "bias":
            continue
        if p.shape != x.shape[-1:] or p.device != x.device or p.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be [{x.shape[-1]}] of x's type or fp32 on its device")


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
                       eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)``; the statistics are fp32, one per row."""
    if x.is_cuda:
        y, mean, rstd = ext().layer_norm_fwd(x, weight, bias, eps)
        return y, mean, rstd
    _check(x, weight, bias)
    f = x.reshape(-1, x.shape[-1]).float()
    mean = f.mean(-1)
    c = f - mean[:, None]
    rstd = torch.rsqrt(c.square().mean(-1) + eps)
    y = c * rstd[:, None] * weight.float() + (0 if bias is None else bias.float())
    return y.to(x.dtype).view(x.shape), mean, rstd


def layer_norm_backward(
    dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
    bias_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, dweight, dbias)`` from the forward's input and statistics; ``dbias``
    has ``bias_dtype`` (the weight's type when None)."""
    bias_dtype = bias_dtype or weight.dtype
    if bias_dtype not in (x.dtype, torch.float32):
        raise ValueError("the bias has x's type or fp32")
    if x.is_cuda:
        launches.add(1)                           # the join of the column sums
        dx, dw, db = ext().layer_norm_bwd(dy, x, weight, mean, rstd, bias_dtype == torch.float32,
                                          err_word(x.device))
        return dx, dw, db
    _check(x, weight, None)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError(f"dy must be like x: {tuple(dy.shape)} {dy.dtype}, {tuple(x.shape)} {x.dtype}")
    rows, gf = x.reshape(-1, x.shape[-1]).float(), dy.reshape(-1, x.shape[-1]).float()
    if mean.shape != (rows.shape[0],) or rstd.shape != mean.shape:
        raise ValueError("mean and rstd must hold one value per row of x")
    n = (rows - mean[:, None]) * rstd[:, None]
    a = gf * weight.float()
    dx = rstd[:, None] * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
    return dx.to(x.dtype).view(x.shape), (gf * n).sum(0).to(weight.dtype), gf.sum(0).to(bias_dtype)


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
        return *refuse_second("layer_norm", (dx, dw, None if ctx.bias_dtype is None else db), dy, x, weight), None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) * rstd * weight + bias`` over the last dimension, differentiable in all three."""
    return _LayerNorm.apply(x, weight, bias, float(eps))
