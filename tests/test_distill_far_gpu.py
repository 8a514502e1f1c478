"""A student whose listed logits stand far above all others: the mass that it leaves outside the list has no place in 32 bits beside the list's, and
its logarithm and its shares still decide the loss and the gradient. Against sums of logarithms in 64 bits, and against differences of them.

Tolerances: a logit over the temperature, or a teacher's less its log-sum, is off by a few units of 2^-24 of its size, and a sum of
exponentials by 1e-5 of itself; both stand in `e`. A probability is off by e of itself, the teacher's rest by e of its mass (as large as the
rest here), a loss by 2 e of itself (and of 1), a gradient by e (q + p) and, outside the list, by 2 e of the token's share of the rest; a bfloat16
gradient by 2^-8 of itself besides."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.test_logit_rows_gpu import BF16, DEV, EPS, F32, ops, rows_at

pytestmark = pytest.mark.gpu


def log_sum_exp(z: np.ndarray) -> float:
    m = z.max() if len(z) else -math.inf
    return m + math.log(np.exp(z - m).sum()) if m > -math.inf else -math.inf


def in_logarithms(x, ids, teacher, log_sum, tau, weight):
    """(loss, gradient, q, p, the others' shares of the rest) of one row; listed tokens stand once."""
    z = np.asarray(x, dtype=np.float64) / tau
    listed = np.zeros(len(z), dtype=bool)
    listed[ids] = True
    log_q = z - log_sum_exp(z)
    log_p = np.asarray(teacher, dtype=np.float64) / tau - log_sum
    p = np.zeros(len(z))
    p[ids] = np.exp(log_p)
    outside = log_sum_exp(z[~listed])
    share = np.where(listed, 0.0, np.exp(z - outside)) if outside > -math.inf else np.zeros(len(z))
    rest_p = max(0.0, 1.0 - p.sum()) if outside > -math.inf else 0.0
    loss = sum(np.exp(lp) * (lp - log_q[i]) for i, lp in zip(ids, log_p) if lp > -math.inf)
    if rest_p > 0:
        loss += rest_p * (math.log(rest_p) - (outside - log_sum_exp(z)))
    q = np.exp(log_q)
    gradient = q * (p.sum() + rest_p) - p - rest_p * share
    return weight * tau**2 * loss, weight * tau * gradient, q, p, share


class Far:
    """Rows whose `k` listed logits lead by about `lead`; the teacher's mass on them is `mass`."""

    def __init__(self, rows, vocab, k, lead, tau, dtype=F32, mass=0.4, seed=0):
        gen = torch.Generator().manual_seed(seed + vocab + k)
        student = torch.randn(rows, vocab, generator=gen)
        self.ids = torch.stack([torch.randperm(vocab, generator=gen)[:k] for _ in range(rows)]).to(torch.int32)
        student.scatter_add_(1, self.ids.long(), torch.full((rows, k), float(lead)))
        self.teacher = torch.randn(rows, k, generator=gen) * min(1.0, tau)
        self.log_sum = (torch.logsumexp(self.teacher.double() / tau, dim=1) - math.log(mass)).float()
        self.weight = 0.5 + torch.rand(rows, generator=gen)
        self.x, self.tau, self.dtype = rows_at(student, dtype, 1, 2), tau, dtype

    def run(self, gradient=True):
        return ops().distill_loss(self.x, self.ids.to(DEV), self.teacher.to(DEV), log_sum=self.log_sum.to(DEV), temperature=self.tau,
                                  weight=self.weight.to(DEV), gradient=gradient)

    def want(self, r, x=None):
        x = self.x[r].double().cpu().numpy() if x is None else x
        return in_logarithms(x, self.ids[r].long().numpy(), self.teacher[r].double().numpy(), float(self.log_sum[r]), self.tau, float(self.weight[r]))

    def check(self, loss, gradient):
        for r in range(self.x.shape[0]):
            want, slopes, q, p, share = self.want(r)
            scale = float(self.weight[r]) * self.tau
            sizes = self.x[r].double().abs().cpu().numpy()
            e = 1e-5 + 8 * EPS * ((sizes[np.isfinite(sizes)].max() + float(self.teacher[r].abs().max())) / self.tau + abs(float(self.log_sum[r])))
            assert float(loss[r]) >= 0
            assert abs(float(loss[r]) - want) <= 2 * e * (scale * self.tau + abs(want)), (float(loss[r]), want)
            if gradient is None:
                continue
            off = np.abs(gradient[r].double().cpu().numpy() - slopes)
            allowed = scale * (e * (q + p) + 2 * e * share) + (2.0**-8 * np.abs(slopes) if self.dtype == BF16 else 0.0)
            assert np.all(off <= allowed + 1e-37), (off - allowed).max()   # (below float32's normal numbers: nothing)


@pytest.mark.parametrize("lead,tau", [(0, 1.0), (60, 1.0), (84, 1.0), (88, 1.0), (95, 1.0), (104, 1.0), (120, 1.0), (200, 1.0), (44, 0.5), (60, 0.5), (9, 0.1),
                                      (14, 0.1), (300, 2.5), (3, 0.01)])
@pytest.mark.parametrize("vocab,k", [(40, 1), (1031, 8), (50257, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_loss_of_a_far_list(vocab, k, lead, tau, dtype):
    case = Far(3, vocab, k, lead, tau, dtype)
    loss, gradient = case.run()
    case.check(loss, gradient)
    case.check(case.run(gradient=False)[0], None)


@pytest.mark.parametrize("vocab,dtype", [(131079, F32), (300007, BF16), (440011, F32)])
def test_distill_loss_of_a_far_list_in_long_rows(vocab, dtype):
    """Rows over several CTAs, and rows that no cluster holds."""
    for lead in (20, 110):
        case = Far(2, vocab, 20, lead, 1.0, dtype)
        case.check(*case.run())
        case.check(case.run(gradient=False)[0], None)


def test_distill_gradient_of_a_far_list_against_differences():
    case = Far(2, 60, 4, 110, 1.0)
    _, gradient = case.run()
    direction = torch.randn(2, 60, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    h = 1e-4
    for r in range(2):
        x, d = case.x[r].double().cpu().numpy(), direction[r].numpy()
        slope = (case.want(r, x + h * d)[0] - case.want(r, x - h * d)[0]) / (2 * h)
        got = float((gradient[r].double().cpu() * direction[r]).sum())
        # h^2 of a third derivative below 10; losses below 200 in 64 bits: 200 * 2^-52 / h; the gradient's numbers, below 1 in all, by 3e-5
        assert abs(got - slope) <= 1e-7 + 1e-9 + 3e-5 * float(direction[r].abs().max()) * 2, (got, slope)


@pytest.mark.parametrize("faint", [-60.0, -86.0, -90.0, -95.0, -99.0, -103.0, -110.0])
@pytest.mark.parametrize("tau", [1.0, 0.1])
@pytest.mark.parametrize("vocab", [64, 50257])
def test_distill_entries_of_hardly_any_mass(faint, tau, vocab):
    """Listed tokens of which the teacher thinks next to nothing (below 32 bits' normal numbers, or nothing in 32 bits at all) and the student does not."""
    case = Far(3, vocab, 6, 0, tau)
    case.teacher[:, 3] = (case.log_sum.double() + faint).float() * tau
    case.teacher[1, 5] = case.teacher[1, 3]
    loss, gradient = case.run()
    case.check(loss, gradient)
    case.check(case.run(gradient=False)[0], None)


@pytest.mark.parametrize("vocab", [40, 50257])
@pytest.mark.parametrize("tail", [True, False])
def test_distill_rows_of_nothing_have_no_loss(vocab, tail):
    """Logits that are all -inf, that hold infinity or NaN, or that no reference reaches: NaN, with entries and without."""
    case = Far(9, vocab, 5, 0, 1.0)
    x = case.x.clone()
    x[0:2] = -math.inf
    x[2:4] = torch.finfo(F32).min
    x[4, 3], x[5, 3] = math.inf, math.nan
    x[6, case.ids[6, 0].item()], x[7, case.ids[7, 0].item()] = math.inf, math.nan
    case.ids[[1, 3, 5]] = -1
    for gradient in (True, False):
        loss, _ = ops().distill_loss(x, case.ids.to(DEV), case.teacher.to(DEV), log_sum=case.log_sum.to(DEV) if tail else None, gradient=gradient)
        # (without the other outcome and without entries nothing is compared: 0)
        assert torch.isnan(loss[:8] if tail else loss[[0, 2, 4, 6, 7]]).all() and torch.isfinite(loss[8])


@pytest.mark.parametrize("mass", [1.002, 1.3])
@pytest.mark.parametrize("vocab", [40, 50257])
def test_distill_lists_of_more_than_the_whole_mass(mass, vocab):
    """A teacher's logits that were rounded after their sum was taken: more than 1 on the list, nothing left beside it."""
    case = Far(3, vocab, 6, 0, 1.0, mass=mass)
    case.check(*case.run())
    case.check(case.run(gradient=False)[0], None)
