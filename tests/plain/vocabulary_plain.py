"""The two ends of a token table in float64: the loss of tokens from hidden rows with its gradients, rows by tokens and their gradient, and how far
sums in 32 bits may be from them."""

from __future__ import annotations

import torch

EPS = 2.0**-24


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


class Loss:
    """Everything about one call: `loss`, `log_sum`, `d_hidden`, `d_table`, and `*_off`, by which a kernel's results may differ.

    A logit is a sum of D products of numbers of 24 bits at most, each exact to 4 units (float32 numbers go in as three terms of eight bits, whose
    smallest products are left out: 2^-24 of a product), added in steps that are off by 2 units (of 2^-24) of what has been added, at most 2 D of
    them: (4 D + 16) units of sum |x w|. The exponentials: the exponent's rounding (a unit of the logits and of the sum's logarithm, times a few) and
    2^-21 for the function and the additions in between of a tile; 1e-5 covers the sums. Gradients: a row's factors dz have the errors
    of two logits in their exponents, and one rounding to the type; sums of K products as above, one rounding of the result."""

    def __init__(self, hidden, table, targets, weight=None, softcap=0.0):
        x, w = hidden.detach().double(), table.detach().double()
        rows, width = x.shape
        vocab = w.shape[0]
        rounding = half_step(hidden.dtype)
        inner = rounding if hidden.dtype is torch.bfloat16 else 4 * EPS   # of dz
        u = x @ w.t()
        z = softcap * torch.tanh(u / softcap) if softcap > 0 else u
        self.z = z
        self.log_sum = torch.logsumexp(z, dim=1)
        held = (targets >= 0) & (targets < vocab)
        a = torch.ones(rows, dtype=torch.float64, device=x.device) if weight is None else weight.double()
        a = torch.where(held, a, 0.0)
        at = targets.clamp(0, vocab - 1).long()[:, None]
        self.loss = torch.where(a != 0, a * (self.log_sum - z.gather(1, at)[:, 0]), 0.0)
        p = torch.exp(z - self.log_sum[:, None])
        dz = p.scatter_add(1, at, torch.full_like(at, -1.0, dtype=torch.float64)) * a[:, None]
        slope = 1 - (z / softcap) ** 2 if softcap > 0 else torch.ones_like(z)
        dz = torch.where(a[:, None] != 0, dz * slope, 0.0)
        counted = torch.where(a[:, None] != 0, x, 0.0)
        self.d_hidden, self.d_table = dz @ w, dz.t() @ counted

        size = (x.abs() @ w.abs().t()).amax(dim=1)
        logit = (4 * width + 16) * EPS * size + 16 * EPS * softcap
        self.log_sum_off = logit + 1e-5 + 16 * EPS * (self.log_sum.abs() + size)
        self.loss_off = a.abs() * 2 * self.log_sum_off
        # a factor: exp's argument is off by the logit's and the sum's error; the rounding; where 1 - p cancels, the 1's rounding
        exponent = torch.expm1(2 * self.log_sum_off)[:, None]
        dz_off = (p * slope * a.abs()[:, None]) * exponent + dz.abs() * inner + 4 * EPS * a.abs()[:, None] * torch.zeros_like(z).scatter(1, at, 1.0)
        if softcap > 0:   # (the slope's error: 2 t times the tanh's, and its own rounding)
            dz_off = dz_off + (p + 0.0).scatter_add(1, at, torch.ones_like(at, dtype=torch.float64)) * a.abs()[:, None] * \
                (2 * (logit / softcap)[:, None] + 16 * EPS)
        dz_off = torch.where(a[:, None] != 0, dz_off, 0.0)
        self.d_hidden_off = dz_off @ w.abs() + (4 * vocab / 8 + 64) * EPS * (dz.abs() @ w.abs()) + rounding * self.d_hidden.abs() + 1e-37
        self.d_table_off = dz_off.t() @ counted.abs() + (4 * rows / 8 + 64) * EPS * (dz.abs().t() @ counted.abs()) + rounding * self.d_table.abs() + 1e-37


def rows_gradient(ids, above, vocab, scale=1.0, into=None):
    """(the table's gradient, by how much the kernel's may differ: a step per addition, one more for the scale, the rounding of the result)."""
    held = (ids >= 0) & (ids < vocab)
    at, rows = ids[held].long(), above.detach().double()[held] * scale
    out = torch.zeros(vocab, above.shape[1], dtype=torch.float64, device=above.device).index_add_(0, at, rows)
    size = torch.zeros_like(out).index_add_(0, at, rows.abs())
    count = torch.zeros(vocab, dtype=torch.float64, device=above.device).index_add_(0, at, torch.ones(len(at), dtype=torch.float64, device=above.device))
    if into is not None:
        out = out + into.double()
        size = size + into.double().abs() * (count > 0)[:, None]
    return out, (count[:, None] + 2) * EPS * size
