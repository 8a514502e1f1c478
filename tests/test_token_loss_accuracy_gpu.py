"""How exact losses of tokens and their gradients are where many rows, long rows or large batches could cost it: against 64 bits, with tolerances derived beside them
(`tests/plain/vocabulary_plain.py` has the operators' own)."""

from __future__ import annotations

import pytest
import torch

from tests.plain.vocabulary_plain import Loss
from tests.test_token_loss_gpu import BF16, DEV, F32, Case, gen, ops

pytestmark = pytest.mark.gpu


def common(c: Case, token: int, share: float) -> Case:
    """One token for a share of the rows, scattered; its neighbours for a few more."""
    hot = torch.rand(len(c.targets), generator=gen(1), device=DEV) < share
    hot[:8] = False
    c.targets[hot] = token
    c.targets[7], c.targets[8], c.targets[9] = token - 1, token + 1, token + 32
    return c


@pytest.mark.parametrize("rows,width,vocab,token,share", [
    (129, 64, 1500, 40, 0.0), (300, 96, 2500, 31, 0.1), (700, 257, 300, 255, 0.5), (1000, 72, 5000, 4000, 0.3), (513, 40, 64, 20, 0.95), (2000, 130, 900, 640, 0.04),
    (70001, 40, 300, 77, 0.2)])
def test_what_rounding_leaves_of_a_tokens_own_factor_is_in_the_tables_gradient(rows, width, vocab, token, share):
    """bfloat16, tokens that the model finds unlikely: a row's factor is nearly all at its own token, a (p - 1). Its rounding, half a step of |a (p - 1)| times the hidden row, is not
    in the table's gradient however many rows there are: the tolerance is the oracle's without it (4 units of 2^-24 in its place)."""
    c = common(Case(rows, width, vocab, BF16, rows, size=0.05), token, share)
    got, want = c.run(), c.plain()
    a = torch.where((c.targets >= 0) & (c.targets < vocab), c.weight.double(), 0.0)
    y = c.targets.clamp(0, vocab - 1).long()
    own = a * torch.expm1(want.z.gather(1, y[:, None])[:, 0] - want.log_sum)
    less = (2.0**-8 - 4 * 2.0**-24) * own.abs()[:, None]
    x = torch.where(a[:, None] != 0, c.hidden.double(), 0.0)
    off = want.d_table_off.index_add(0, y, -less * x.abs())
    assert torch.all((got[3].double() - want.d_table).abs() <= off)
    assert all(torch.equal(one, other) for one, other in zip(got, c.run()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width,vocab", [(4096, 768, 50257), (2047, 1600, 10007)])
def test_steps_of_training(rows, width, vocab, dtype):
    common(Case(rows, width, vocab, dtype, rows), 13, 0.1).check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("sign", [-1, 1])
def test_targets_far_beyond_the_cap(rows, dtype, sign):
    """Row i learns token i, whose raw logit u is 3 to 12 caps below (above) 0: a factor is (p - 1 at a row's own token, p elsewhere) times the slope 1 - tanh(u / cap)^2, which has to be right relative to
    itself however small it is. u is one exact product; u / cap and the exponent 2 |u / cap| log2 e are rounded five times, so that exp(2 |u / cap|) is off by 2 |u / cap| times five units of 2^-24, and a few
    units come from the functions and the slope's products: (12 |u / cap| + 64) units of a factor. The rest as the oracle has it, each times the slope: what the logarithm of the sum leaves of a p, the 1's
    rounding, the factors' (bfloat16), the sums' and the result's. (Above 0 a token's p of all rows nearly cancel its 1, so that these are most of it.)"""
    cap, vocab, width = 6.0, 600, 8
    table = torch.randn(vocab, width, generator=gen(2), device=DEV)
    far = sign * cap * (3 + 9 * torch.rand(rows, generator=gen(3), device=DEV))
    table[:rows, 0] = far
    hidden = torch.zeros(rows, width, device=DEV)
    hidden[:, 0] = 1.0
    c = Case(1, width, vocab, dtype)
    c.hidden, c.table, c.softcap, c.weight = hidden.to(dtype), table.to(dtype), cap, None
    c.targets = torch.arange(rows, dtype=torch.int32, device=DEV)
    _, _, _, d_table = c.run()
    want = c.plain()
    x = c.table[:rows, 0].double().abs() / cap
    z = want.z[:, :rows]   # [row, token]
    p, slope, own = torch.exp(z - want.log_sum[:, None]), 1 / torch.cosh(c.table[:rows, 0].double() / cap) ** 2, torch.eye(rows, device=DEV, dtype=torch.float64)
    dz = (p - own).abs() * slope
    dz_off = p * slope * torch.expm1(2 * want.log_sum_off)[:, None] + own * slope * 4 * 2.0**-24 + dz * ((12 * x + 64) * 2.0**-24 + (2.0**-8 if dtype is BF16 else 0.0))
    off = dz_off.sum(0) + (4 * rows / 8 + 64) * 2.0**-24 * dz.sum(0) + (2.0**-8 if dtype is BF16 else 2.0**-24) * want.d_table[:rows, 0].abs()
    assert torch.all((d_table[:rows, 0].double() - ((p - own) * slope).sum(0)).abs() <= off)


def test_sums_over_very_many_rows():
    """Tensor cores cut every addition of 16 products by up to a unit of 2^-24 of the sum, towards zero, so that sums of one sign are off by as many units as they have additions: 524,288 rows have
    32,768 of them. Sums of 32,768 rows at most are made there (2,048 units at most), and joined rounded to nearest. The mean over a table's gradient of 31 x 1,024 numbers of the error relative to each: of
    the cuts 2^-13; of the results' and factors' rounding, 2^-8 / sqrt(3) each for one number, 6 deviations of the mean; of the probabilities 1e-5, as the oracle has it."""
    rows, width, vocab = 524288, 1024, 32
    hidden = torch.empty(rows, width, dtype=BF16, device=DEV)
    for i in range(0, rows, 65536):   # positive; columns all over a binade, so that their roundings differ
        hidden[i: i + 65536] = (0.5 + torch.rand(65536, width, generator=gen(i), device=DEV)) * 2 ** torch.linspace(0, 1, width, device=DEV)
    table = (torch.randn(vocab, width, generator=gen(5), device=DEV) / 32).to(BF16)
    targets = torch.zeros(rows, dtype=torch.int32, device=DEV)
    _, log_sum = ops().token_loss(hidden, table, targets)
    _, d_table = ops().token_loss_gradient(hidden, table, targets, log_sum, hidden_gradient=False)
    ops().raise_on_device_error(DEV)
    want = torch.zeros(vocab, width, dtype=torch.float64, device=DEV)
    for i in range(0, rows, 65536):
        x = hidden[i: i + 65536].double()
        want += torch.softmax(x @ table.double().t(), 1).t() @ x
    error = ((d_table.double() - want) / want)[1:]   # (token 0's: p - 1)
    assert abs(error.mean().item()) <= 2.0**-13 + 6 * 2 * 2.0**-8 / 3**0.5 / error.numel() ** 0.5 + 1e-5


@pytest.mark.parametrize("rows", [64, 256])
def test_the_gradients_logits_are_the_losses(rows):
    """Rows of 16,384 positive numbers, logits near 40: products added in one sum on the tensor cores would leave them 1,024 cuts of up to 2^-24 of 40 too low (2.4e-3), pieces of 512 (few rows: 256) 32 (16) of them.
    A factor exp(z - log_sum) takes its z from pieces of 1,024 (few rows: of the loss's): the mean over all factors, relative, differs by what cuts differ by (64 in place of 32: 32 units of 2^-24 of 48; few
    rows: none) and what the sum's logarithm (near 48, rounded three times:
    1.2e-5), exponent and function (5e-6) are rounded to; the factors' own rounding, 6 deviations of the mean; the cuts of 256 rows' sums (16 units of 2^-24)."""
    width, vocab = 16384, 2000
    hidden = (1 + torch.rand(rows, width, generator=gen(6), device=DEV)).to(BF16)
    table = ((0.5 + torch.rand(vocab, width, generator=gen(7), device=DEV)) * (40 / 1.5 / width)).to(BF16)
    targets = torch.zeros(rows, dtype=torch.int32, device=DEV)
    loss, log_sum = ops().token_loss(hidden, table, targets)
    _, d_table = ops().token_loss_gradient(hidden, table, targets, log_sum, hidden_gradient=False)
    want = Loss(hidden, table, targets)
    error = ((d_table.double() - want.d_table) / want.d_table)[1:]
    cuts = 32 * 2.0**-24 * 48 if rows > 128 else 0.0
    assert abs(error.mean().item()) <= cuts + 1.7e-5 + 6 * 2.0**-8 / 3**0.5 / ((vocab - 1) * rows) ** 0.5 + 6 * 2.0**-8 / 3**0.5 / error.numel() ** 0.5 + 16 * 2.0**-24


@pytest.mark.parametrize("rows,width,vocab", [(300, 16, 1200003), (9000, 40, 50001), (20000, 72, 3000)])
def test_one_gradient_alone_of_sorted_rows(rows, width, vocab):
    """bfloat16, several pieces of the vocabulary or several segments of rows: what a gradient is made from lies where the piece before left its own; alone it is what it is beside the other."""
    c = common(Case(rows, width, vocab, BF16, rows), vocab // 2, 0.1)
    c.targets[10:16] = torch.tensor([0, vocab - 1, vocab // 3, 524287 % vocab, 524288 % vocab, 1048575 % vocab], dtype=torch.int32, device=DEV)
    both = c.run()
    for _ in range(3):
        assert torch.equal(c.run(hidden_gradient=False)[3], both[3]) and torch.equal(c.run(table_gradient=False)[2], both[2])
    if rows * vocab < 4e8:
        c.check()
