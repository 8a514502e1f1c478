"""Rows masked with a low number instead of -inf: -1e10, -1e30, the type's lowest. Such numbers are too large for a reference that sums are taken
against (neighbours of 2^31 in 32 bits lie 256 apart), and weigh nothing beside others.

Tolerances: as for rows masked with -inf, whose results they have to equal within 1e-5 of the sums."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_logit_rows_gpu import BF16, DEV, EPS, F32, ops, random_logits, rows_at

pytestmark = pytest.mark.gpu
LOW = [-7e9, -1e10, -7e12, -1e30, "lowest"]


def masked(rows, vocab, low, dtype, seed, keep):
    """Logits of which `keep` a row are left, and the same with -inf in place of the others."""
    low = torch.finfo(dtype).min if low == "lowest" else low
    gen = torch.Generator().manual_seed(seed)
    left = torch.zeros(rows, vocab, dtype=torch.bool)
    left.scatter_(1, torch.stack([torch.randperm(vocab, generator=gen)[:keep] for _ in range(rows)]), True)
    x = random_logits(rows, vocab, seed).to(dtype).float()
    return (rows_at(torch.where(left, x, value), dtype, 1, 2) for value in (torch.tensor(low), torch.tensor(-math.inf)))


@pytest.mark.parametrize("rows,vocab", [(3, 200), (700, 200), (3, 4000), (2, 50257), (200, 30011)])
@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0, 3.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_logits_of_rows_masked_with_a_low_number(rows, vocab, low, tau, dtype):
    x, none = masked(rows, vocab, low, dtype, vocab, 11)
    got, want = ops().top_logits(x, 9, temperature=tau), ops().top_logits(none, 9, temperature=tau)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.all((got[2] - want[2]).abs() <= 1e-5 + 4 * EPS * want[2].abs())


@pytest.mark.parametrize("low", [*LOW, -3e9, 3e9, 1e30, "highest"])
@pytest.mark.parametrize("vocab", [200, 4000, 50257])
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_top_logits_of_rows_far_from_nothing(low, vocab, tau):
    """Rows of one number alone, as far from 0 as 32 bits go: the logarithm of the sum is that number over the temperature, to its own precision."""
    low = {"lowest": torch.finfo(F32).min, "highest": torch.finfo(F32).max}.get(low, low)
    x = torch.full((2, vocab), low, device=DEV)
    values, ids, log_sum = ops().top_logits(x, 5, temperature=tau)
    assert torch.all(values == x[0, 0]) and ids[0].tolist() == [0, 1, 2, 3, 4]
    want = float(x[0, 0]) / tau + math.log(vocab)
    assert torch.all((log_sum.double() - want).abs() <= 1e-5 + 4 * EPS * abs(want)) or abs(float(x[0, 0]) / tau * 1.4427) > 3.4e38


@pytest.mark.parametrize("rows,vocab,k", [(3, 200, 5), (2, 50257, 9), (2, 131079, 7), (700, 3000, 6)])
@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0, 3.0])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_loss_of_students_masked_with_a_low_number(rows, vocab, k, low, tau, tail, dtype):
    for keep in (k, k + 30):   # the listed tokens alone; some others beside them
        x, none = masked(rows, vocab, low, dtype, vocab + keep, keep)
        left = torch.topk(none.float(), keep, dim=1).indices
        order = torch.argsort(torch.rand(rows, keep, generator=torch.Generator().manual_seed(1)), dim=1).to(DEV)
        ids = torch.gather(left, 1, order)[:, :k].to(torch.int32).contiguous()
        teacher = torch.randn(rows, k, generator=torch.Generator().manual_seed(2)).to(DEV)
        log_sum = torch.logsumexp(teacher / tau, dim=1) + 0.5 if tail else None
        for gradient in (True, False):
            loss, slopes = ops().distill_loss(x, ids, teacher, log_sum=log_sum, temperature=tau, gradient=gradient)
            want, its = ops().distill_loss(none, ids, teacher, log_sum=log_sum, temperature=tau, gradient=gradient)
            assert torch.isfinite(want).all() and torch.all((loss - want).abs() <= 1e-5 * tau * tau * (1 + want.abs()))
            if gradient:
                assert torch.all((slopes.float() - its.float()).abs() <= 2e-5 * tau + (2.0**-7 * its.float().abs() if dtype == BF16 else 0))
