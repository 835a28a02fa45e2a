"""Embedding lookup with a scale and a trained table (csrc/embedding_grad.cu).

``embedding(ids, table, scale=s)`` is ``s * table[ids]`` (one rounding),
differentiable in ``table`` (once: a second derivative raises);
``embedding_grad`` is its gradient for callers that run their backward by hand,
written whole or added to a gradient that is there (a table that is also the
vocabulary projection).

The gradient sorts the tokens by id and adds each row's tokens in fp32 in token
order: the result does not depend on timing, whatever the repetitions, and is
rounded once.  ``padding_idx`` names a row that gets no gradient.  An id outside
the table gives a NaN row and no gradient, and ``check_errors`` raises.

Tables and gradients are bf16, fp16 or fp32.  On the CPU the same functions
compute with PyTorch operations.  The reference's table is frozen
(src/graspo/backends/graspoflow/models/qwen3/model.py:262-269).
"""

from __future__ import annotations

import torch

from graspo_b200.ops._ext import err_word, ext, launches
from graspo_b200.ops._second import refuse_second

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_NO_ID = -(1 << 63)


def _check_padding(padding_idx: int, vocab: int) -> None:
    if not 0 <= padding_idx < vocab:
        raise ValueError(f"padding_idx {padding_idx} is outside the table of {vocab} rows")


# The kernels' own checks, for tensors that do not reach them.
def _check_ids(ids: torch.Tensor, device: torch.device, vocab: int, padding_idx: int | None) -> torch.Tensor:
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32, not {ids.dtype}")
    if ids.device != device:
        raise ValueError("ids must be on the device of the table")
    if padding_idx is not None:
        _check_padding(padding_idx, vocab)
    flat = ids.reshape(-1).long()
    if bool(((flat < 0) | (flat >= vocab)).any()):
        raise IndexError("a token id is outside the table")
    return flat


def _check_table(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2 or 0 in t.shape or t.dtype not in _TYPES:
        raise ValueError(f"{name} must be a bf16, fp16 or fp32 matrix, not {tuple(t.shape)} {t.dtype}")


def _lookup(ids: torch.Tensor, table: torch.Tensor, scale: float, padding_idx: int | None) -> torch.Tensor:
    if table.is_cuda:
        if padding_idx is not None:
            _check_padding(padding_idx, table.shape[0])
        return ext().embed_fwd(ids, table, scale, err_word(table.device))
    _check_table(table, "table")
    flat = _check_ids(ids, table.device, table.shape[0], padding_idx)
    return (table[flat].float() * scale).to(table.dtype).view(*ids.shape, -1)


def embedding_grad(dy: torch.Tensor, ids: torch.Tensor, vocab: int, *, scale: float = 1.0,
                   padding_idx: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient [vocab, H] of ``embedding``'s table from ``dy`` [*ids.shape, H].

    Without ``out`` it is a new tensor of ``dy``'s type.  With ``out`` [vocab, H]
    (contiguous, any of the three types) the touched rows are added to it in
    fp32 and rounded to its type; the others are not read."""
    if dy.is_cuda:
        if padding_idx is not None:
            _check_padding(padding_idx, vocab)
        n = ids.numel()
        launches.add((n > 1024) + (out is None) + (n >= 128) + (n >= 4096) + 2)  # sort, merge, places, groups, rows
        return ext().embed_bwd(dy, ids, vocab, out, scale, _NO_ID if padding_idx is None else padding_idx,
                               err_word(dy.device))
    if dy.shape[:-1] != ids.shape or dy.dim() < 1 or dy.shape[-1] == 0:
        raise ValueError(f"dy {tuple(dy.shape)} must have one row per id {tuple(ids.shape)}")
    if dy.dtype not in _TYPES or vocab < 1:
        raise ValueError(f"dy must be bf16, fp16 or fp32, not {dy.dtype}, and the table needs a row")
    H = dy.shape[-1]
    if out is not None:
        _check_table(out, "out")
        if out.shape != (vocab, H) or out.device != dy.device or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous [{vocab}, {H}] on the device of dy")
    flat, rows = _check_ids(ids, dy.device, vocab, padding_idx), dy.reshape(-1, H)
    keep = torch.ones_like(flat, dtype=torch.bool) if padding_idx is None else flat != padding_idx
    total = torch.zeros(vocab, H, dtype=torch.float32) if out is None else out.float()
    total.index_add_(0, flat[keep], rows[keep].float() * scale)
    return total.to(dy.dtype) if out is None else out.copy_(total)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.dtype, ctx.scale, ctx.padding = table.shape[0], table.dtype, scale, padding_idx
        return _lookup(ids, table, scale, padding_idx)

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        grad = embedding_grad(dy, ids, ctx.vocab, scale=ctx.scale, padding_idx=ctx.padding)
        return None, *refuse_second("embedding", (grad,), dy), None, None


def embedding(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * table[ids]`` [*ids.shape, H], differentiable in ``table`` (a dense gradient)."""
    if torch.is_grad_enabled() and table.requires_grad:
        return _Embedding.apply(ids, table, float(scale), padding_idx)
    return _lookup(ids, table, scale, padding_idx)
