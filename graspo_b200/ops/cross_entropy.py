"""Cross entropy of hidden states against a vocabulary projection, without the logits.

``linear_cross_entropy(h, weight, targets)`` is ``F.cross_entropy(h @ weight^T,
targets)`` for hidden states ``h`` [..., H] and a projection ``weight`` [V, H],
as an autograd function of both (on the GPU differentiable once: a second
derivative raises); ``linear_cross_entropy_grads`` returns the loss and both
gradients at once for callers that run their backward by hand (as
``models/fused.py`` does).

* ``targets`` equal to ``ignore_index`` take no part: loss 0, gradient 0, and
  what their rows of ``h`` hold is never read into a sum.  Their rows cost no
  products either: the rest is compacted first.
* ``reduction``: ``"mean"`` over the trained tokens (0 where there are none),
  ``"sum"``, or ``"none"`` (one fp32 loss per token).
* A target outside the vocabulary gives a NaN loss and no gradient, and
  ``check_errors`` raises.

On the GPU ``h`` and ``weight`` are bf16, any H, V and number of tokens; logits
and sums are fp32, the gradients bf16.  The logits exist one tile at a time;
the backward remakes them in pieces of the vocabulary (csrc/cross_entropy.cu).
On the CPU the same functions compute with PyTorch operations.

The reference keeps the logits of the whole batch (src/graspo/core/sft_loss.py:12-34)
and trains no vocabulary projection; ``ops/head.py`` is this framework's
selected-token log-prob of a frozen one.
"""

from __future__ import annotations

import torch

from graspo_b200.ops._ext import err_word, ext, launches
from graspo_b200.ops._second import refuse_second

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


# The kernels' own checks, for tensors that do not reach them.
def _check(h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, reduction: str, piece: int) -> None:
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(REDUCTIONS)}, not {reduction!r}")
    if weight.dim() != 2 or h.dim() < 1 or h.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"h [..., H] and weight [V, H] do not match: {tuple(h.shape)}, {tuple(weight.shape)}")
    if targets.shape != h.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} must have one entry per row of h {tuple(h.shape)}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets must be int64 or int32, not {targets.dtype}")
    if piece < 0 or piece % 256:
        raise ValueError("piece must be a multiple of 256")
    if h.device != weight.device or h.device != targets.device:
        raise ValueError("h, weight and targets must be on one device")


def _torch_loss(h, weight, targets, ignore_index, reduction):
    """The same definition with PyTorch operations (CPU), differentiable."""
    t = targets.reshape(-1).long()
    live = t != ignore_index
    if bool(((t < 0) | (t >= weight.shape[0]))[live].any()):
        raise IndexError("a target is outside the vocabulary")
    rows = h.reshape(-1, h.shape[-1])[live].float()
    loss = -torch.log_softmax(rows @ weight.float().T, -1).gather(1, t[live][:, None])[:, 0]
    if reduction == "none":
        return torch.zeros(t.shape, dtype=torch.float32, device=h.device).masked_scatter(live, loss).view(targets.shape)
    return loss.sum() / max(1, loss.numel()) if reduction == "mean" else loss.sum()


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, targets, ignore_index, reduction, piece):
        (loss, *state), count = ext().ce_forward(h, weight, targets, ignore_index, REDUCTIONS[reduction],
                                                 ctx.needs_input_grad[1], err_word(h.device))
        launches.add(count - 1)
        ctx.save_for_backward(weight, *state)
        ctx.shape, ctx.tokens, ctx.reduction, ctx.piece = h.shape, targets.numel(), reduction, piece
        return loss

    @staticmethod
    def backward(ctx, g):
        weight, hc, state, h_edge = ctx.saved_tensors
        (dh, dw), count = ext().ce_backward(hc, state, weight, ctx.tokens, g.float().contiguous().view(-1),
                                            REDUCTIONS[ctx.reduction], ctx.needs_input_grad[0],
                                            ctx.needs_input_grad[1], ctx.piece, err_word(hc.device))
        launches.add(count - 1)
        dh, dw = refuse_second("linear_cross_entropy", (None if dh is None else dh.view(ctx.shape), dw),
                               g, weight, h_edge)
        return dh, dw, None, None, None, None


_kernel_loss = _LinearCrossEntropy.apply


def linear_cross_entropy(h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", piece: int = 0) -> torch.Tensor:
    """Cross entropy of ``h @ weight^T`` against ``targets`` (fp32), differentiable in ``h`` and ``weight``.

    ``piece``: vocabulary columns per piece of the backward (a multiple of 256;
    0 takes as many as 256 MiB of softmax gradients hold, at least 256: 512 bytes a
    token, so split calls of more than half a million tokens)."""
    if h.is_cuda and reduction in REDUCTIONS:
        return _kernel_loss(h, weight, targets, int(ignore_index), reduction, int(piece))
    _check(h, weight, targets, reduction, piece)
    return _torch_loss(h, weight, targets, ignore_index, reduction)


def linear_cross_entropy_grads(
    h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, grad: torch.Tensor | None = None,
    ignore_index: int = -100, reduction: str = "mean", weight_grad: bool = True, piece: int = 0,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """``(loss, dh, dweight)`` of ``linear_cross_entropy`` in one call, without an autograd graph.

    ``grad`` is the upstream gradient of the result (one value; one per token
    for ``reduction="none"``; ones when absent).  ``weight_grad=False`` leaves
    the projection's gradient out (a frozen head)."""
    if h.is_cuda and reduction in REDUCTIONS:
        if grad is not None:
            grad = grad.detach().float().contiguous()
        (loss, dh, dw), count = ext().ce_grads(h, weight, targets, grad, ignore_index, REDUCTIONS[reduction],
                                               weight_grad, piece, err_word(h.device))
        launches.add(count - 1)
        return loss, dh, dw
    _check(h, weight, targets, reduction, piece)
    if grad is not None and (grad.numel() != (targets.numel() if reduction == "none" else 1)
                             or grad.device != h.device):
        raise ValueError("grad must have one value, or one per token for reduction='none', on the device of h")
    hl, wl = h.detach().requires_grad_(True), weight.detach().requires_grad_(True)
    with torch.enable_grad():
        loss = _torch_loss(hl, wl, targets, ignore_index, reduction)
        up = torch.ones_like(loss) if grad is None else grad.float().view(loss.shape)
        dh, dw = torch.autograd.grad(loss, (hl, wl), up)
    return loss.detach(), dh, dw if weight_grad else None
