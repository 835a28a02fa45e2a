"""Second derivatives of operators whose backward is a kernel: refused, never left out.

What a kernel returns carries no graph.  Under ``create_graph=True`` the gradients
that it made would therefore be constants to a second derivative, and a term made
of them would drop out of a larger loss without a word.  ``refuse_second`` joins
them to the tensors that they depend on through a node that raises.

(``torch.autograd.function.once_differentiable`` does so only where the upstream
gradient requires one, and joins its node to nothing, so that
``torch.autograd.grad`` for named inputs walks past it.)
"""

from __future__ import annotations

import torch


class _Refuse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, count, *tensors):
        ctx.set_materialize_grads(False)
        ctx.name, ctx.inputs = name, 2 + len(tensors)
        return tensors[:count]

    @staticmethod
    def backward(ctx, *grads):
        if all(g is None for g in grads):
            return (None,) * ctx.inputs
        raise RuntimeError(f"{ctx.name} has no second derivative: its gradients are differentiable no further")


def refuse_second(name: str, grads: tuple, *depends: torch.Tensor | None) -> tuple:
    """``grads`` (some may be None) as a backward returns them; differentiating them raises."""
    if not torch.is_grad_enabled():
        return grads
    return _Refuse.apply(name, len(grads), *grads, *depends)
