"""Global gradient norm over many tensors, and clipping by it (csrc/grad_clip.cu).

``grad_norm(grads)`` is the 2-norm of all values together; ``clip_grad_norm_``
scales them by ``min(1, max_norm / (norm + 1e-6))``, in place or into other
tensors (bf16 gradients into an optimizer's fp32 buffer, say), and returns the
norm before clipping.  Neither waits for the GPU: the norm stays on the device
and the second kernel reads it there.

The coefficient and its treatment of non-finite norms are those of the flat
buffer's optimizer and of ``torch.nn.utils.clip_grad_norm_`` (reference:
qwen35_36/training.py:435-441): a NaN norm makes every value NaN, an infinite
one makes the finite values 0.  ``max_norm=0`` clips nothing, as in ``FlatAdamW``.
The sum does not depend on timing.  Gradients are bf16, fp16 or fp32, mixed as
they come.  On the CPU the same functions compute with PyTorch operations.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from graspo_b200.ops._ext import ext, launches

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_PER_LAUNCH = 896


def _list(tensors: Sequence[torch.Tensor]) -> list[torch.Tensor]:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _check(grads: list[torch.Tensor], out: list[torch.Tensor]) -> None:
    """The kernels' own checks, for tensors that do not reach them."""
    for g in grads + out:
        if g.dtype not in _TYPES or not g.is_contiguous() or g.device != grads[0].device:
            raise ValueError("gradients and outputs must be contiguous bf16, fp16 or fp32 tensors on one device")
    if any(o.shape != g.shape for o, g in zip(out, grads)):
        raise ValueError("outputs must have the gradients' shapes")


def _norm_torch(grads: list[torch.Tensor]) -> torch.Tensor:
    total = torch.zeros((), dtype=torch.float64)
    for g in grads:
        total += g.detach().double().square().sum()
    return total.sqrt().float()


def _device(grads: list[torch.Tensor]) -> torch.device:
    return grads[0].device if grads else torch.device("cuda" if torch.cuda.is_available() else "cpu")


def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """2-norm over all values of ``grads`` (a 0-dim fp32 tensor on their device; 0 without any)."""
    grads = _list(grads)
    dev = _device(grads)
    if dev.type != "cuda":
        _check(grads, [])
        return _norm_torch(grads)
    launches.add(-(-len(grads) // _PER_LAUNCH))
    return ext().grad_norm(grads, dev.index if dev.index is not None else torch.cuda.current_device())


def clip_grad_norm_(grads: Sequence[torch.Tensor], max_norm: float,
                    out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """Scale ``grads`` to a global norm of at most ``max_norm``; the norm before it.

    With ``out`` (one tensor per gradient, of its size and any of the three
    types) the scaled values go there and ``grads`` stay as they are.  What is
    written must not overlap: a tensor that is there twice is a race."""
    grads = _list(grads)
    out = None if out is None else _list(out)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative: {max_norm}")
    if out is not None and len(out) != len(grads):
        raise ValueError(f"{len(out)} outputs for {len(grads)} gradients")
    dev = _device(grads)
    if dev.type != "cuda":
        _check(grads, out or [])
        norm = _norm_torch(grads)
        coef = (max_norm / (norm + 1e-6)).clamp(max=1.0) if max_norm > 0 else torch.ones(())
        with torch.no_grad():
            for g, o in zip(grads, grads if out is None else out):
                o.copy_(g.float() * coef)
        return norm
    launches.add(-(-len(grads) // _PER_LAUNCH))
    return ext().grad_clip(grads, out or [], max_norm, dev.index if dev.index is not None else torch.cuda.current_device())
