"""The two ends of a token table, for training with torch's gradients: the rows that tokens look up, and the loss of tokens from hidden rows. The loss keeps no
logits [N, V]: the backward pass makes them again, as factors of up to 512 MB at a time (a piece of the vocabulary, or all of it where it fits), with the factors that come down from above.
(A step that is to be captured into a graph asks for its gradients with `torch.autograd.grad`, or calls the operators themselves: while an eager graph over the same
parameters lives, torch itself cannot capture a `backward()` that adds to their `.grad`.)"""

from __future__ import annotations

import torch

from ..kernels import ops


def _tokens(t: torch.Tensor, vocab: int) -> torch.Tensor:
    """int32; wider numbers that name no token stay such."""
    return t if t.dtype is torch.int32 else t.clamp(-1, vocab).to(torch.int32)


def _contiguous_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() != 2 or t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


class _TokenLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, table, targets, weight, softcap):
        loss, log_sum = ops.token_loss(hidden.detach(), table.detach(), targets, weight=weight, softcap=softcap)
        ctx.save_for_backward(hidden, table, targets, weight, log_sum)
        ctx.softcap = softcap
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, above):
        hidden, table, targets, weight, log_sum = ctx.saved_tensors
        factor = (above.to(torch.float32) if weight is None else above * weight).contiguous()
        d_hidden, d_table = ops.token_loss_gradient(hidden, table, targets, log_sum, weight=factor, softcap=ctx.softcap,
                                                    hidden_gradient=ctx.needs_input_grad[0], table_gradient=ctx.needs_input_grad[1])
        return d_hidden, d_table, None, None, None


def token_loss(hidden: torch.Tensor, table: torch.Tensor, targets: torch.Tensor, *, weight: torch.Tensor | None = None, softcap: float = 0.0) -> torch.Tensor:
    """weight * (minus the log-probability of the target) of every row of `hidden` [..., D], float32 [...], with gradients for `hidden` and `table` [V, D]
    (`ops.token_loss` says what they are; `targets` [...] may be int64, `weight` is float32 [...]). There is no gradient for `weight`: one that asks for it is
    refused (`detach()` it)."""
    if weight is not None and torch.is_grad_enabled() and weight.requires_grad:
        raise ops.KernelError("token_loss: weight asks for a gradient and there is none: detach() it")
    if targets.dtype not in (torch.int32, torch.int64):
        raise ops.KernelError(f"token_loss: targets must be int32 or int64, got {targets.dtype}")
    if hidden.dim() < 1 or hidden.shape[:-1] != targets.shape or (weight is not None and weight.shape != targets.shape):
        raise ops.KernelError(f"token_loss: hidden rows {tuple(hidden.shape)}, targets {tuple(targets.shape)}" +
                              (f" and weights {tuple(weight.shape)}" if weight is not None else "") + " do not fit")
    if table.dim() != 2:
        raise ops.KernelError(f"token_loss: table must have 2 dimensions, got shape {tuple(table.shape)}")
    if hidden.shape[-1] < 1:
        raise ops.KernelError(f"token_loss: hidden rows {tuple(hidden.shape)} have no numbers")
    rows = hidden.reshape(-1, hidden.shape[-1])
    loss = _TokenLoss.apply(_contiguous_rows(rows), _contiguous_rows(table), _tokens(targets, table.shape[0]).reshape(-1).contiguous(),
                            None if weight is None else weight.reshape(-1).contiguous(), float(softcap))
    return loss.view(targets.shape)


class _TokenRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, out_dtype):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.vocab, ctx.dtype = scale, table.shape[0], table.dtype
        return ops.token_rows(ids, table.detach(), scale=scale, out_dtype=out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, above):
        (ids,) = ctx.saved_tensors
        if ctx.vocab == 0:   # (all rows were zeros)
            return None, above.new_zeros((0, above.shape[1]), dtype=ctx.dtype), None, None
        return None, ops.token_rows_gradient(ids, _contiguous_rows(above), ctx.vocab, scale=ctx.scale, out_dtype=ctx.dtype), None, None


def token_rows(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """scale * table[ids], of ids (int32 or int64) of any shape: [..., D], with a gradient for `table` [V, D], added in one order
    (`ops.token_rows` and `ops.token_rows_gradient` say what they are). A token outside [0, V) gets zeros and gives nothing."""
    if ids.dtype not in (torch.int32, torch.int64):
        raise ops.KernelError(f"token_rows: ids must be int32 or int64, got {ids.dtype}")
    if table.dim() != 2:
        raise ops.KernelError(f"token_rows: table must have 2 dimensions, got shape {tuple(table.shape)}")
    rows = _TokenRows.apply(_tokens(ids, table.shape[0]).reshape(-1).contiguous(), _contiguous_rows(table), float(scale), out_dtype)
    return rows.view(*ids.shape, table.shape[1])


__all__ = ["token_loss", "token_rows"]
