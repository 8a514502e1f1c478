"""A student's loss against a teacher's top logits, for training with torch's gradients: the kernels behind `kernels.ops.distill_loss` compute loss
and gradient in one pass over the logits, so the backward pass only scales the gradient by what comes down from above, and not even
that where it is 1 (give a mean's 1 / n as `weight`, and sum). Where the graph is kept (`retain_graph`) the scaled gradient is written apart, and
every backward pass over it starts from the same one."""

from __future__ import annotations

import torch

from ..kernels import ops


# Whether the backward pass that runs keeps its graph, in which what a node has saved is wanted again. (Where torch cannot say: it may.)
_graph_is_kept = getattr(torch._C._autograd, "_get_current_graph_task_keep_graph", lambda: True)


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, log_sum, temperature, weight):
        wanted = ctx.needs_input_grad[0]
        loss, gradient = ops.distill_loss(logits.detach(), ids, teacher, log_sum=log_sum, temperature=temperature, weight=weight, gradient=wanted)
        if wanted:
            ctx.save_for_backward(gradient)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, above):
        (gradient,) = ctx.saved_tensors
        return ops.scale_rows(gradient, above.to(torch.float32).contiguous(), in_place=not _graph_is_kept()), None, None, None, None, None


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *, log_sum: torch.Tensor | None = None, temperature: float = 1.0,
                 weight: torch.Tensor | None = None) -> torch.Tensor:
    """weight * temperature^2 * KL(teacher || student) of every row, float32 [R], with a gradient for `logits` [R, V] (float32 or bfloat16). `ids`
    and `teacher` [R, K] are a teacher's top logits and `log_sum` [R] the logarithm of its sum of exponentials at this temperature, as
    `ops.top_logits` and the `teach` command give them; without `log_sum` the teacher's probabilities are spread over its K tokens alone. There is
    no gradient for them nor for `weight`: one that asks for it is refused (`detach()` it)."""
    if torch.is_grad_enabled():
        for name, t in (("teacher", teacher), ("log_sum", log_sum), ("weight", weight)):
            if t is not None and t.requires_grad:
                raise ops.KernelError(f"distill_loss: {name} asks for a gradient and there is none: detach() it")
    return _DistillLoss.apply(logits, ids, teacher, log_sum, temperature, weight)


__all__ = ["distill_loss"]
