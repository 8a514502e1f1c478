"""The distillation loss in torch's graphs: a graph that is kept gives the same gradients every time. On the CPU above kernels replaced by their
definitions (in place where they are), and with the kernels themselves."""

from __future__ import annotations

import pytest
import torch

from research_2_b200.kernels import ops
from research_2_b200.sampling import distill

ROWS, VOCAB = 3, 37


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        def distill_loss(logits, ids, teacher, *, log_sum=None, temperature=1.0, weight=None, gradient=True, out=None):
            with torch.enable_grad():
                x = logits.detach().clone().requires_grad_()
                p = torch.softmax(teacher / temperature, dim=1)
                log_q = torch.log_softmax(x / temperature, dim=1)
                loss = weight * temperature**2 * (p * (torch.log(p) - torch.gather(log_q, 1, ids.long()))).sum(1)
                slopes = torch.autograd.grad(loss.sum(), x)[0]
            return loss.detach(), slopes if gradient else None

        def scale_rows(x, factors, *, in_place=True):
            scaled = x * factors.reshape(-1, 1)
            if not in_place:
                return scaled
            x.data.copy_(scaled)   # (past torch's version counter, as a kernel writes)
            return x

        monkeypatch.setattr(ops, "distill_loss", distill_loss)
        monkeypatch.setattr(ops, "scale_rows", scale_rows)
    return request.param


def student(device):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(ROWS, VOCAB, generator=gen).to(device).requires_grad_()
    values, ids = torch.topk(torch.randn(ROWS, VOCAB, generator=gen), 5, dim=1)
    weight = torch.tensor([1.0, 0.5, 2.0], device=device)
    loss = distill.distill_loss(x, ids.to(torch.int32).to(device), values.to(device), temperature=2.0, weight=weight)
    x64 = x.detach().double().cpu().requires_grad_()
    p = torch.softmax(values.double() / 2.0, dim=1)
    want = weight.double().cpu() * 4 * (p * (torch.log(p) - torch.gather(torch.log_softmax(x64 / 2.0, dim=1), 1, ids))).sum(1)
    rows = torch.stack([torch.autograd.grad(want[i], x64, retain_graph=True)[0][i] for i in range(ROWS)])
    return x, loss, rows


def close(got: torch.Tensor, want: torch.Tensor) -> bool:
    # numbers of at most 4 of a softmax in 32 bits
    return torch.allclose(got.double().cpu(), want, rtol=1e-5, atol=1e-5)


def test_a_kept_graph_gives_the_same_gradient_again(device):
    x, loss, rows = student(device)
    first = torch.autograd.grad(loss.mean(), x, retain_graph=True)[0]
    kept = first.clone()
    second = torch.autograd.grad(loss.mean(), x, retain_graph=True)[0]
    assert close(first, rows / 3) and close(second, rows / 3) and torch.equal(first, kept)
    whole = torch.autograd.grad(loss.sum(), x, retain_graph=True)[0]
    whole.zero_()   # (a caller's own)
    last = torch.autograd.grad((loss * 3).sum(), x)[0]
    assert close(last, rows * 3) and torch.equal(first, kept) and torch.equal(second, kept)
    with pytest.raises(RuntimeError):
        loss.sum().backward()


def test_rows_gradients_one_by_one(device):
    x, loss, rows = student(device)
    for i in range(ROWS):
        got = torch.autograd.grad(loss[i], x, retain_graph=True)[0]
        want = torch.zeros_like(rows)
        want[i] = rows[i]
        assert close(got, want)


def test_gradients_add_up_in_the_leaf(device):
    x, loss, rows = student(device)
    loss.sum().backward(retain_graph=True)
    loss.mean().backward(retain_graph=True)
    (loss * torch.tensor([0.0, 1.0, -2.0], device=device)).sum().backward()
    assert close(x.grad, rows * (4 / 3) + rows * torch.tensor([[0.0], [1.0], [-2.0]]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,offset", [(1, 0), (7, 3), (2049, 1), (50257, 0)])
def test_scale_rows_into_new_rows(dtype, vocab, offset):
    buf = torch.randn(5, vocab + offset + 2, device="cuda:0").to(dtype)
    x, before = buf[:, offset: offset + vocab], buf.clone()
    for factors in (torch.tensor([1.0, 0.5, -3.0, 0.0, 1.7], device="cuda:0"), torch.ones((), device="cuda:0")):
        got = ops.scale_rows(x, factors, in_place=False)
        assert got.data_ptr() != x.data_ptr() and got.dtype == dtype
        assert torch.equal(got, (x.float() * factors.reshape(-1, 1)).to(dtype)) and torch.equal(buf, before)
    assert ops.scale_rows(x[:0], torch.ones(1, device="cuda:0"), in_place=False).shape == (0, vocab)


@pytest.mark.parametrize("name", ["teacher", "log_sum", "weight"])
def test_what_has_no_gradient_is_refused_where_it_asks_for_one(name):
    given = {"teacher": torch.randn(2, 3), "log_sum": torch.randn(2), "weight": torch.ones(2)}
    given[name].requires_grad_()
    x, ids = torch.randn(2, 9, requires_grad=True), torch.tensor([[0, 1, 2]] * 2, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match=f"{name} asks for a gradient"):
        distill.distill_loss(x, ids, given.pop("teacher"), **given)
