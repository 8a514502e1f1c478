"""Operators on rows of logits against statements in 64 bits: sizes around a piece, a CTA's slice and a cluster's, both types, rows at every
alignment, masks that leave nothing, infinities, NaN, ties, lists with nothing in them, rows far into a large buffer.

Tolerances: a float32 result of a few operations is off by a few units of 2^-24 of the largest number in them, a bfloat16 result by another
2^-9 of itself. A sum of exponentials of up to 50,257 terms is added in at most some 100 steps by a thread and 16 levels above that:
1e-5 of itself; a loss is a sum of weights times logarithms (below 100 in these cases), so 1e-5 times the largest of them."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.plain import logits_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 2.0**-24
F32, BF16 = torch.float32, torch.bfloat16


def ops():
    from research_2_b200.kernels import ops as o

    return o


def rows_at(values: torch.Tensor, dtype, offset: int = 0, pad: int = 0) -> torch.Tensor:
    """The values as a view that starts `offset` places into rows of `offset + V + pad`; what lies around them is NaN."""
    r, v = values.shape
    buf = torch.full((r, offset + v + pad), float("nan"), dtype=dtype, device=DEV)
    buf[:, offset: offset + v] = values.to(dtype)
    return buf[:, offset: offset + v]


def random_logits(rows: int, vocab: int, seed: int, scale: float = 3.0) -> torch.Tensor:
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(rows, vocab, generator=gen) * scale


def i32(x) -> torch.Tensor:
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def f32(x) -> torch.Tensor:
    return torch.tensor(np.asarray(x), dtype=F32, device=DEV)


def pack_mask(allowed: np.ndarray, spare_words: int = 0) -> torch.Tensor:
    m, v = allowed.shape
    bits = np.zeros((m, (v + 31) // 32 + spare_words, 32), dtype=np.uint32)
    bits.reshape(m, -1)[:, :v] = allowed
    return torch.from_numpy((bits << np.arange(32, dtype=np.uint32)).sum(axis=2).astype(np.uint32).view(np.int32)).to(DEV)


def close(got: torch.Tensor, want: np.ndarray, size: float, dtype) -> None:
    """Equal infinities and NaN; else within 8 units of `size`, and of the result's own rounding."""
    got = got.detach().double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    allowed = 8 * EPS * size + (2.0**-8 * np.abs(want[fine]) if dtype == BF16 else 0.0)
    assert np.all(np.abs(got[fine] - want[fine]) <= allowed), np.abs(got[fine] - want[fine]).max()


# ---- adjust_logits ------------------------------------------------------------------------------

class Adjust:
    """Random rows with histories, biases and masks, and what they make of the logits."""

    def __init__(self, rows, vocab, cap, n_biases, seed, dtype=F32, offset=0, pad=0):
        rng = np.random.default_rng(seed)
        self.x = rows_at(random_logits(rows, vocab, seed), dtype, offset, pad)
        self.dtype, self.rows, self.vocab = dtype, rows, vocab
        wide = max(1, vocab // 3)
        self.history = rng.integers(-3, wide + 3 if vocab > 6 else vocab + 3, size=(rows + 2, max(cap, 1))).astype(np.int32)
        self.history[-1, :] = vocab - 1
        self.slots = rng.permutation(rows + 2)[:rows]
        self.lengths = rng.integers(0, cap + 1, size=rows)
        self.lengths[0] = cap
        self.prompts = rng.integers(0, self.lengths + 1)
        self.rho, self.presence, self.frequency = rng.uniform(0.5, 2.0, rows), rng.uniform(-1, 1, rows), rng.uniform(-0.5, 0.5, rows)
        counts = rng.integers(0, n_biases + 1, size=rows)
        counts[-1] = n_biases
        self.start = np.concatenate([[0], np.cumsum(counts)])
        self.bias_ids = rng.integers(-2, vocab + 2, size=self.start[-1])
        self.bias_values = rng.uniform(-3, 3, size=self.start[-1])
        self.allowed = rng.random((max(1, rows // 2), vocab)) < rng.choice([0.02, 0.5, 0.98], size=(max(1, rows // 2), 1))
        self.mask_rows = rng.integers(-1, len(self.allowed), size=rows)
        self.mask_rows[-1] = 0

    def arguments(self):
        return dict(history=i32(self.history), slots=i32(self.slots), lengths=i32(self.lengths), prompt_lengths=i32(self.prompts),
                    repetition=f32(self.rho), presence=f32(self.presence), frequency=f32(self.frequency), bias_start=i32(self.start),
                    bias_ids=i32(self.bias_ids), bias_values=f32(self.bias_values), mask=pack_mask(self.allowed, 1), mask_rows=i32(self.mask_rows))

    def want(self):
        out = []
        as32 = lambda a: np.asarray(a, dtype=np.float32).astype(np.float64)  # noqa: E731
        for r in range(self.rows):
            held = self.history[self.slots[r], : self.lengths[r]].tolist()
            a, b = self.start[r], self.start[r + 1]
            out.append(plain.adjust_row(
                self.x[r].double().cpu().numpy(), held[: self.prompts[r]], held[self.prompts[r]:], as32(self.rho)[r], as32(self.presence)[r],
                as32(self.frequency)[r], list(zip(self.bias_ids[a:b].tolist(), as32(self.bias_values)[a:b])),
                self.allowed[self.mask_rows[r]] if self.mask_rows[r] >= 0 else None))
        return np.stack(out)


ADJUST = [(1, 1, 3, 2), (2, 5, 9, 7), (3, 31, 0, 0), (3, 33, 40, 5), (2, 1031, 300, 64), (4, 4096, 1, 1), (2, 4095, 700, 33), (3, 4101, 129, 300),
          (1, 8200, 5000, 10), (2, 50257, 1000, 300)]


@pytest.mark.parametrize("rows,vocab,cap,n_biases", ADJUST)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adjust_logits(rows, vocab, cap, n_biases, dtype):
    for offset, pad in ((0, 0), (1, 2), (3, 5)):
        case = Adjust(rows, vocab, cap, n_biases, vocab + cap, dtype, offset, pad)
        before = case.x.clone()
        got = ops().adjust_logits(case.x, **case.arguments())
        assert got.dtype == dtype and got.shape == case.x.shape
        want = case.want()
        size = 60.0 + cap   # of a logit and its penalties
        close(got, want, size, dtype)
        assert torch.equal(case.x, before)
        again = ops().adjust_logits(case.x, **case.arguments(), out=torch.empty(rows, vocab, dtype=dtype, device=DEV))
        assert torch.equal(again, got)
        inside = ops().adjust_logits(case.x, **case.arguments(), out=case.x)
        assert inside.data_ptr() == case.x.data_ptr() and torch.equal(inside, got)


@pytest.mark.parametrize("vocab,cap", [(3000, 16384), (40001, 40000)])
def test_adjust_logits_long_histories(vocab, cap):
    """Histories longer than the counts that 16 bits hold, one token standing in almost all of one."""
    case = Adjust(2, vocab, cap, 5, 11, F32, 1, 2)
    case.history[case.slots[0], 100:] = 17
    case.lengths[0], case.prompts[0] = cap, 30
    got = ops().adjust_logits(case.x, **case.arguments())
    want = case.want()
    fine = np.isfinite(want)
    off = np.abs(got.double().cpu().numpy()[fine] - want[fine])
    # the penalty of a token that stands c times: c * frequency in float32
    assert np.array_equal(np.isfinite(got.cpu().numpy()), fine) and np.all(off <= 8 * EPS * (60 + np.abs(want[fine])))


def test_adjust_logits_writes_nothing_but_its_rows():
    case = Adjust(3, 1031, 50, 9, 5, BF16, offset=3, pad=6)
    out = rows_at(torch.zeros(3, 1031), BF16, 1, 4)
    buf = out._base
    around = buf.isnan().sum()
    ops().adjust_logits(case.x, **case.arguments(), out=out)
    assert buf.isnan().sum() == around


def test_adjust_logits_parts_alone_and_nothing_at_all():
    x = rows_at(random_logits(4, 777, 3), F32)
    assert torch.equal(ops().adjust_logits(x), x)
    history = i32([[5, 5, 9, 776], [0, 0, 0, 0], [1, 2, 3, 4], [7, 7, 7, 7]])
    got = ops().adjust_logits(x, history=history, lengths=i32([4, 0, 3, 4]), frequency=f32([0.5, 0.5, 0.5, 0.25]))
    want = np.stack([plain.adjust_row(x[r].double().cpu().numpy(), (), h, frequency=f) for r, (h, f) in
                     enumerate([([5, 5, 9, 776], 0.5), ([], 0.5), ([1, 2, 3], 0.5), ([7] * 4, 0.25)])])
    close(got, want, 20.0, F32)
    allowed = np.zeros((2, 777), dtype=bool)
    allowed[1, 700] = True
    got = ops().adjust_logits(x, mask=pack_mask(allowed), mask_rows=i32([0, 1, -1, 5]))
    assert torch.all(got[0] == -math.inf) and got[1, 700] == x[1, 700] and torch.isinf(got[1]).sum() == 776
    assert torch.equal(got[2:], x[2:])
    params = [torch.ones(4, device=DEV), i32([1, 0, 0, 0]), i32([0] * 4), i32([0] * 4), i32([0] * 4)]
    drawn = ops().sample(got, *params)
    assert drawn[0] == 0 and drawn[1] == 700   # a row that nothing is left of answers 0


def test_adjust_logits_infinities_and_nan():
    x = torch.zeros(1, 40, device=DEV)
    x[0, :6] = torch.tensor([math.inf, -math.inf, math.nan, math.nan, 1.0, -1.0])
    allowed = np.ones((1, 40), dtype=bool)
    allowed[0, [3, 7]] = False
    got = ops().adjust_logits(x, history=i32([[0, 1, 2, 4, 5]]), lengths=i32([5]), repetition=f32([2.0]), mask=pack_mask(allowed))
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and math.isnan(got[0, 2]) and got[0, 3] == -math.inf
    assert got[0, 4] == 0.5 and got[0, 5] == -2.0 and got[0, 7] == -math.inf


def test_adjust_logits_adds_biases_of_one_token_in_order():
    x = torch.zeros(2, 100, device=DEV)
    values = np.float32([1e8, 1.0, -1e8, 3.0] * 20)
    ids = [7, 7, 7, 9] * 20
    got = ops().adjust_logits(x, bias_start=i32([0, 80, 80]), bias_ids=i32(ids), bias_values=f32(values))
    sums = np.zeros(100, dtype=np.float32)
    for i, v in zip(ids, values):
        sums[i] += v
    assert np.array_equal(got[0].cpu().numpy(), sums) and torch.all(got[1] == 0)


# ---- top_logits ---------------------------------------------------------------------------------

def check_top(x: torch.Tensor, k: int, temperature: float = 1.0):
    values, ids, log_sum = ops().top_logits(x, k, temperature=temperature)
    assert values.dtype == F32 and ids.dtype == torch.int32 and log_sum.dtype == F32
    for r in range(x.shape[0]):
        want_v, want_i, want_s = plain.top_row(x[r].double().cpu().numpy(), k, temperature)
        assert ids[r].tolist() == list(want_i), r
        assert np.array_equal(values[r].double().cpu().numpy(), want_v, equal_nan=True)
        got = float(log_sum[r])
        if math.isfinite(want_s):
            assert abs(got - want_s) <= 1e-5 + 4 * EPS * abs(want_s), (r, got, want_s)
        else:
            assert got == want_s or (math.isnan(got) and math.isnan(want_s))
    return values, ids, log_sum


@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (2, 9, 9), (5, 33, 4), (3, 256, 256), (2, 300, 255), (4, 1031, 20), (2, 4096, 64), (1, 12289, 128),
                                          (3, 16385, 3), (2, 50257, 5), (2, 50257, 256), (1, 131080, 100), (1, 300007, 17)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_logits(rows, vocab, k, dtype):
    for offset, pad in ((0, 0), (1, 0), (5, 3)) if vocab < 60000 else ((1, 2),):
        check_top(rows_at(random_logits(rows, vocab, vocab + k), dtype, offset, pad), k, 1.0 + k / 100)


@pytest.mark.parametrize("rows", [1, 40, 300, 700])
def test_top_logits_at_several_numbers_of_rows(rows):
    x = rows_at(random_logits(rows, 3001, rows), BF16, 1)
    values, ids, _ = ops().top_logits(x, 30)
    order = torch.argsort(x.float(), dim=1, descending=True, stable=True)[:, :30]
    assert torch.equal(ids.long(), order) and torch.equal(values, torch.gather(x.float(), 1, order))


@pytest.mark.parametrize("vocab", [700, 50257, 140003])
def test_top_logits_of_equal_values(vocab):
    x = torch.zeros(4, vocab)
    x[1] = torch.arange(vocab) % 3       # thousands of equal values at the edge of the list
    x[2, vocab // 2:] = -math.inf
    x[3] = -math.inf
    x[0, 11], x[0, 500] = -0.0, 1e-30
    check_top(rows_at(x, F32, 1), 64)
    check_top(rows_at(x, BF16, 3), 200)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_logits_of_many_rows_some_of_equal_values(dtype):
    """Several rows a CTA, those that are gone over (equal values, few numbers) next to others, in every order."""
    rows, vocab, k = 900, 9001, 40
    x = random_logits(rows, vocab, 6).to(dtype).to(DEV)
    kind = torch.randint(0, 5, (rows,), generator=torch.Generator().manual_seed(2)).to(DEV)
    kind[100:130], kind[450:600] = 0, 1
    x[kind == 0] = 1.5
    x[kind == 1, 20:] = -math.inf
    x[kind == 2] = (torch.arange(vocab, device=DEV) % 7).to(dtype)
    values, ids, _ = ops().top_logits(x, k)
    order = torch.argsort(x.float(), dim=1, descending=True, stable=True)[:, :k]
    assert torch.equal(ids.long(), order) and torch.equal(values, torch.gather(x.float(), 1, order))


@pytest.mark.parametrize("rows", [2, 37, 400])
@pytest.mark.parametrize("vocab,k", [(1300, 256), (2049, 129), (2561, 256), (5120, 200), (10241, 256), (40001, 256), (90003, 256)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_logits_of_many_candidates(rows, vocab, k, dtype):
    """Long lists, whose candidates fill many runs, from one row over several CTAs to several rows a CTA; every third row has few values."""
    x = random_logits(rows, vocab, vocab + rows)
    x[::3] = torch.round(x[::3] * 4)
    x = rows_at(x, dtype, 1, 2)
    values, ids, _ = ops().top_logits(x, k)
    order = torch.argsort(x.float(), dim=1, descending=True, stable=True)[:, :k]
    assert torch.equal(ids.long(), order) and torch.equal(values, torch.gather(x.float(), 1, order))


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("vocab,k", [(1, 1), (9, 9), (129, 128), (257, 5), (511, 200), (1020, 64), (1029, 128), (2044, 256), (2053, 100), (4080, 33), (4105, 64), (8190, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_logits_of_short_rows(rows, vocab, k, dtype):
    """A warp's rows, 128 threads' rows and the first that they do not hold; some of few values, of few numbers, of none."""
    x = random_logits(rows, vocab, vocab + 3 * rows)
    x[::4] = torch.round(x[::4])
    x[1::16, vocab // 3:] = -math.inf
    x[2::16] = 0.5
    x = rows_at(x, dtype, 3, 1)
    values, ids, log_sum = ops().top_logits(x, k, temperature=1.5)
    order = torch.argsort(x.float(), dim=1, descending=True, stable=True)[:, :k]
    assert torch.equal(ids.long(), order) and torch.equal(values, torch.gather(x.float(), 1, order))
    want = torch.logsumexp(x.double() / 1.5, dim=1)
    assert torch.all((log_sum == want) | ((log_sum.double() - want).abs() <= 1e-5 + 4 * EPS * want.abs()))   # (-inf equals -inf)
    if rows > 3:
        holed = x.clone()
        holed[::5] = math.nan
        holed[1::5, :: 2] = math.nan
        check_top(holed[:12], k)


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_top_logits_of_rows_in_order(order):
    x = torch.linspace(-20, 20, 50257)[None].repeat(2, 1)
    check_top(rows_at(x if order == "rising" else x.flip(1), F32, 1), 256)


def test_top_logits_infinities_and_nan():
    x = random_logits(6, 5000, 8)
    x[0, 77] = math.inf
    x[1, 5] = math.nan
    x[2] = math.nan
    x[3, 100:] = -math.inf
    x[4, 4990:] = math.nan
    x[5, 3] = x[5, 4999] = math.inf
    check_top(rows_at(x, F32, 3), 128)


# ---- distill_loss -------------------------------------------------------------------------------

class Distill:
    def __init__(self, rows, vocab, k, seed, dtype=F32, tail=True, temperature=1.0, offset=0, pad=0, gap=1.0):
        gen = torch.Generator().manual_seed(seed)
        teacher = torch.randn(rows, vocab, generator=gen) * 3
        student = teacher + gap * torch.randn(rows, vocab, generator=gen)
        self.values, ids = torch.topk(teacher, k, dim=1)
        self.ids = ids.to(torch.int32)
        if rows > 1 and k > 1:
            self.ids[1, k // 2:] = -1     # a row with fewer entries
        self.log_sum = torch.logsumexp(teacher.double() / temperature, dim=1).float() if tail else None
        self.weight = 0.5 + torch.rand(rows, generator=gen)
        self.x, self.tau, self.dtype = rows_at(student, dtype, offset, pad), temperature, dtype

    def run(self, gradient=True, out=None, x=None):
        return ops().distill_loss(self.x if x is None else x, self.ids.to(DEV), self.values.to(DEV),
                                  log_sum=None if self.log_sum is None else self.log_sum.to(DEV), temperature=self.tau,
                                  weight=self.weight.to(DEV), gradient=gradient, out=out)

    def want(self, x=None):
        x = self.x if x is None else x
        both = [plain.distill_row(x[r].double().cpu().numpy(), self.ids[r].tolist(), self.values[r].double().tolist(),
                                  None if self.log_sum is None else float(self.log_sum[r]), self.tau, float(self.weight[r]))
                for r in range(x.shape[0])]
        return np.array([b[0] for b in both]), np.stack([b[1] for b in both])

    def check(self, loss, gradient):
        want_loss, want = self.want()
        scale = self.weight.double().numpy() * self.tau**2
        finite = np.isfinite(want_loss)
        got = loss.double().cpu().numpy()
        assert np.array_equal(got[~finite], want_loss[~finite])
        off = np.abs(got[finite] - want_loss[finite])
        assert np.all(off <= 1e-5 * scale[finite] * (1 + np.abs(want_loss[finite]))), off.max()
        if gradient is None:
            return
        # q and p are off by 1e-5 of themselves; where q's mass is small outside the list, what it is divided by adds 4e-6 / rest
        z = self.x.double().cpu().numpy() / self.tau
        q = np.exp(z - z.max(axis=1, keepdims=True))
        q /= q.sum(axis=1, keepdims=True)
        for r in range(z.shape[0]):
            listed = [i for i in self.ids[r].tolist() if 0 <= i < z.shape[1]]
            p = np.zeros(z.shape[1])
            p[listed] = 1.0
            rest = max(q[r][p == 0].sum(), 1e-30)
            at = 1e-5 * (q[r] + (p * 1.0)) + 4e-6 * np.minimum(1.0, q[r] / rest)
            allowed = scale[r] / self.tau * at + (2.0**-8 * np.abs(want[r]) if self.dtype == BF16 else 0.0)
            off = np.abs(gradient[r].double().cpu().numpy() - want[r])
            assert np.all(off <= allowed), (r, (off / allowed).max())


DISTILL = [(1, 2, 1), (2, 5, 5), (3, 33, 8), (2, 257, 256), (5, 1031, 8), (3, 4096, 64), (2, 16389, 100), (3, 50257, 64), (1, 131080, 33), (1, 300007, 9)]


@pytest.mark.parametrize("rows,vocab,k", DISTILL)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tail", [True, False])
def test_distill_loss(rows, vocab, k, dtype, tail):
    for offset, pad, tau in ((0, 0, 1.0), (1, 2, 2.5)) if vocab < 60000 else ((3, 0, 2.0),):
        case = Distill(rows, vocab, k, vocab + k, dtype, tail, tau, offset, pad)
        before = case.x.clone()
        loss, gradient = case.run()
        assert loss.dtype == F32 and gradient.dtype == dtype and gradient.shape == case.x.shape
        case.check(loss, gradient)
        assert torch.equal(case.x, before)
        alone, none = case.run(gradient=False)
        assert none is None   # (a kernel of its own, which adds in another order)
        case.check(alone, None)
        apart = torch.empty(rows, vocab, dtype=dtype, device=DEV)
        assert torch.equal(case.run(out=apart)[1], gradient)
        loss_in, inside = case.run(out=case.x)
        assert inside.data_ptr() == case.x.data_ptr() and torch.equal(inside, gradient) and torch.equal(loss_in, loss)


@pytest.mark.parametrize("vocab,dtype", [(440011, F32), (880007, BF16)])
def test_distill_loss_of_rows_that_no_cluster_holds(vocab, dtype):
    case = Distill(2, vocab, 9, 1, dtype, True, 2.0, 1, 0)
    loss, gradient = case.run()
    case.check(loss, gradient)
    inside = case.run(out=case.x)
    assert torch.equal(inside[0], loss) and torch.equal(inside[1], gradient)


def test_distill_lists_that_name_a_token_twice():
    """The gradient counts every entry; nothing else is promised of such a list."""
    case = Distill(2, 3001, 6, 2, F32, False, 1.0)
    case.ids[:, 3] = case.ids[:, 0]
    loss, gradient = case.run()
    want = case.want()[1]
    assert torch.isfinite(loss).all() and np.all(np.abs(gradient.double().cpu().numpy() - want) <= 1e-5)


@pytest.mark.parametrize("rows", [1, 20, 150, 400])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_loss_at_several_numbers_of_rows(rows, dtype):
    case = Distill(rows, 2003, 12, rows, dtype, True, 1.5, offset=1)
    case.check(*case.run())


@pytest.mark.parametrize("tail", [True, False])
def test_distill_gradient_against_differences(tail):
    case = Distill(4, 701, 16, 9, F32, tail, 1.7)
    _, gradient = case.run()
    gen = torch.Generator().manual_seed(1)
    direction = torch.randn(4, 701, generator=gen, dtype=torch.float64)
    slope = (gradient.double().cpu() * direction).sum(dim=1).numpy()
    h = 1e-5
    x = case.x.double().cpu()
    up, down = case.want(x + h * direction)[0], case.want(x - h * direction)[0]
    # the differences of 64-bit losses: h^2 of a third derivative below 1e3, 1e-15 / h of rounding
    assert np.all(np.abs((up - down) / (2 * h) - slope) <= 1e-6 + 2e-5 * (gradient.double().cpu().abs() * direction.abs()).sum(dim=1).numpy() + 1e-5)
    # and of the kernel's own float32 losses: 1e-6 of rounding over 2 h, h^2 / 6 of the third derivative
    h = 2e-2
    up = case.run(gradient=False, x=(x + h * direction).float().to(DEV))[0]
    down = case.run(gradient=False, x=(x - h * direction).float().to(DEV))[0]
    assert np.all(np.abs(((up - down) / (2 * h)).double().cpu().numpy() - slope) <= 1e-2 * (1 + np.abs(slope)))


def test_distill_rows_that_weigh_nothing_are_not_read():
    case = Distill(6, 1031, 8, 3, F32, True, 2.0)
    case.weight[[0, 4]] = 0.0
    case.x[0], case.x[4] = math.nan, math.inf
    loss, gradient = case.run()
    assert torch.all(loss[[0, 4]] == 0) and torch.all(gradient[[0, 4]] == 0)
    keep = [1, 2, 3, 5]
    part = Distill(6, 1031, 8, 3, F32, True, 2.0)
    part.x, part.ids, part.values, part.weight, part.log_sum = case.x[keep], case.ids[keep], case.values[keep], case.weight[keep], case.log_sum[keep]
    part.check(loss[keep], gradient[keep])


@pytest.mark.parametrize("tail", [True, False])
def test_distill_rows_without_entries_and_masked_students(tail):
    case = Distill(5, 600, 6, 4, F32, tail, 1.0)
    case.ids[0] = -1
    if tail:
        case.log_sum[0] = 3.0
    case.values[2, 3] = -math.inf          # a listed token that the teacher forbids
    x = case.x.cpu()
    x[3, case.ids[3, 1]] = -math.inf       # the student forbids what the teacher wants
    x[4, 5:400] = -math.inf                # a masked student
    for i in case.ids[4].tolist():
        x[4, i] = 1.0
    case.x = x.to(DEV)
    loss, gradient = case.run()
    assert loss[3] == math.inf and torch.isfinite(gradient).all()
    if not tail:
        assert loss[0] == 0 and torch.all(gradient[0] == 0)
    case.check(loss, gradient)


def test_distill_lists_that_leave_no_other_token():
    case = Distill(2, 16, 16, 5, F32, True, 1.0)
    case.ids[1] = torch.arange(16, dtype=torch.int32)
    case.check(*case.run())
    wide = Distill(1, 64, 8, 6, F32, True, 1.0)
    x = torch.full((1, 64), -math.inf)
    x[0, wide.ids[0].long()] = torch.randn(8, generator=torch.Generator().manual_seed(0))
    wide.x = x.to(DEV)
    loss, gradient = wide.run()
    assert torch.isfinite(loss).all()
    wide.check(loss, gradient)


def test_distill_entries_outside_the_table_and_rows_of_nothing():
    case = Distill(3, 100, 7, 8, F32, False, 1.0)
    case.ids[0, 2], case.ids[0, 5], case.ids[2, 0] = 100, -7, 2**31 - 1
    x = case.x.clone()
    x[1] = -math.inf
    case.x = x
    loss, gradient = case.run()
    assert math.isnan(float(loss[1]))
    part = Distill(3, 100, 7, 8, F32, False, 1.0)
    part.x, part.ids, part.values, part.weight = x[[0, 2]], case.ids[[0, 2]], case.values[[0, 2]], case.weight[[0, 2]]
    part.check(loss[[0, 2]], gradient[[0, 2]])


# ---- all three ----------------------------------------------------------------------------------

def test_logit_rows_far_into_a_buffer():
    vocab, far = 1031, 2**31 + 5
    buf = torch.empty(far + vocab, dtype=BF16, device=DEV)
    x = torch.as_strided(buf, (2, vocab), (far, 1))
    x.copy_(random_logits(2, vocab, 2))
    near = x.contiguous()
    a, b = ops().top_logits(x, 9), ops().top_logits(near, 9)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    ids, values = b[1], b[0] + 0.25
    loss, gradient = ops().distill_loss(near, ids, values, temperature=2.0)
    far_loss, far_gradient = ops().distill_loss(x, ids, values, temperature=2.0)
    assert torch.equal(loss, far_loss) and torch.equal(gradient, far_gradient)
    arguments = dict(history=i32([[3, 4], [5, 6]]), lengths=i32([2, 1]), presence=f32([1.0, 2.0]))
    want = ops().adjust_logits(near, **arguments)
    assert torch.equal(ops().adjust_logits(x, **arguments, out=x), want)


def test_logit_rows_of_no_rows_and_other_streams():
    nothing = torch.empty(0, 50, device=DEV)
    assert ops().adjust_logits(nothing).shape == (0, 50)
    assert [t.shape[0] for t in ops().top_logits(nothing, 3)] == [0, 0, 0]
    loss, gradient = ops().distill_loss(nothing, torch.empty(0, 2, dtype=torch.int32, device=DEV), torch.empty(0, 2, device=DEV))
    assert loss.shape == (0,) and gradient.shape == (0, 50)
    x = rows_at(random_logits(30, 50257, 1), F32)
    want = ops().top_logits(x, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x * 1.0
        got = ops().top_logits(y, 8)
        loss, gradient = ops().distill_loss(y, got[1], got[0], log_sum=got[2], out=y)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = ops().distill_loss(x, want[1], want[0], log_sum=want[2])
    assert torch.equal(loss, again[0]) and torch.equal(gradient, again[1])


def test_logit_rows_refusals():
    o = ops()
    x = torch.zeros(3, 40, device=DEV)
    ids, values = torch.zeros(3, 4, dtype=torch.int32, device=DEV), torch.zeros(3, 4, device=DEV)
    word = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    refused = [
        lambda: o.adjust_logits(x.cpu()),
        lambda: o.adjust_logits(x.half()),
        lambda: o.adjust_logits(x[0]),
        lambda: o.adjust_logits(x.t()),
        lambda: o.adjust_logits(x[:1].expand(3, 40)),
        lambda: o.adjust_logits(x, out=x.bfloat16()),
        lambda: o.adjust_logits(x, out=torch.zeros(3, 41, device=DEV)),
        lambda: o.adjust_logits(torch.zeros(200, device=DEV)[:120].view(3, 40), out=torch.as_strided(x, (3, 40), (39, 1))),
        lambda: o.adjust_logits(x, history=word),
        lambda: o.adjust_logits(x, history=word.long(), lengths=i32([0] * 3)),
        lambda: o.adjust_logits(x, history=word, lengths=i32([0] * 2)),
        lambda: o.adjust_logits(x, history=word[:2], lengths=i32([0] * 3)),
        lambda: o.adjust_logits(x, repetition=f32([1.0] * 3)),
        lambda: o.adjust_logits(x, history=word, lengths=i32([0] * 3), repetition=f32([1.0] * 3).double()),
        lambda: o.adjust_logits(x, bias_start=i32([0] * 4)),
        lambda: o.adjust_logits(x, bias_start=i32([0] * 3), bias_ids=i32([0]), bias_values=f32([0.0])),
        lambda: o.adjust_logits(x, bias_start=i32([0] * 4), bias_ids=i32([0]), bias_values=f32([])),
        lambda: o.adjust_logits(x, mask=word[:, :1]),
        lambda: o.adjust_logits(x, mask=word[:2]),
        lambda: o.adjust_logits(x, mask=word.float(), mask_rows=i32([0] * 3)),
        lambda: o.top_logits(x, 0),
        lambda: o.top_logits(x, 41),
        lambda: o.top_logits(torch.zeros(1, 400, device=DEV), 257),
        lambda: o.top_logits(x, 3, temperature=0.0),
        lambda: o.top_logits(x, 3, temperature=math.nan),
        lambda: o.top_logits(x.half(), 3),
        lambda: o.top_logits(x.cpu(), 3),
        lambda: o.distill_loss(x, ids.long(), values),
        lambda: o.distill_loss(x, ids, values.bfloat16()),
        lambda: o.distill_loss(x, ids[:2], values[:2]),
        lambda: o.distill_loss(x, ids, values[:, :3]),
        lambda: o.distill_loss(x, ids[:, :0], values[:, :0]),
        lambda: o.distill_loss(x, torch.zeros(3, 257, dtype=torch.int32, device=DEV), torch.zeros(3, 257, device=DEV)),
        lambda: o.distill_loss(x, ids, values, temperature=-1.0),
        lambda: o.distill_loss(x, ids, values, log_sum=f32([0.0])),
        lambda: o.distill_loss(x, ids, values, weight=f32([0.0] * 3).double()),
        lambda: o.distill_loss(x, ids, values, gradient=False, out=x),
        lambda: o.distill_loss(x.double(), ids, values),
    ]
    for i, call in enumerate(refused):
        before = o.launch_count()
        with pytest.raises(o.KernelError):
            call()
        assert o.launch_count() == before, i


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [301, 9001])
def test_distill_many_rows_some_of_no_weight(vocab, dtype):
    """More rows than run at a time: each group of CTAs walks over several, rows of no weight among them, the same bits as one by one."""
    rows, k = 2500, 9
    gen = torch.Generator().manual_seed(vocab)
    x = rows_at(torch.randn(rows, vocab, generator=gen) * 3, dtype, 1)
    values, ids, log_sum = ops().top_logits(rows_at(torch.randn(rows, vocab, generator=gen) * 3, F32), k)
    weight = torch.rand(rows, generator=gen).to(DEV)
    weight[torch.rand(rows, generator=gen).to(DEV) < 0.4] = 0.0
    weight[700:1400] = 0.0
    loss, gradient = ops().distill_loss(x, ids, values, log_sum=log_sum, weight=weight)
    for part in (slice(0, 40), slice(690, 720), slice(1390, 1440), slice(2460, 2500)):
        one, its = ops().distill_loss(x[part], ids[part], values[part], log_sum=log_sum[part], weight=weight[part])
        assert torch.equal(one, loss[part]) and torch.equal(its, gradient[part])
    q = torch.softmax(x.double(), dim=1)
    p = torch.exp(values.double() - log_sum.double()[:, None])
    target = torch.zeros_like(q).scatter_(1, ids.long(), p)
    listed = target > 0
    rest, rest_p = torch.where(listed, 0.0, q).sum(1, keepdim=True), (1 - p.sum(1, keepdim=True)).clamp(min=0)
    want = weight.double()[:, None] * (q - target - torch.where(listed, 0.0, rest_p * q / rest))
    off = (gradient.double() - want).abs()
    assert torch.all(off <= 1e-5 * (q + p.amax(1, keepdim=True) * listed) + 4e-6 * q / rest + (2.0**-8 * want.abs() if dtype == BF16 else 0))


@pytest.mark.parametrize("rows,vocab,k", [(700, 257, 3), (900, 1000, 20), (700, 4001, 64), (650, 12007, 9), (1300, 33, 5)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_of_many_short_rows_is_that_of_few(rows, vocab, k, dtype):
    """More rows than there are places take other numbers of threads; a row's loss and gradient are those of a call on a few rows."""
    gen = torch.Generator().manual_seed(rows)
    x = rows_at(random_logits(rows, vocab, rows), dtype, 1, 2)
    values, ids, log_sum = ops().top_logits(rows_at(torch.randn(rows, vocab, generator=gen) * 3, F32), k)
    weight = torch.rand(rows, generator=gen).to(DEV)
    weight[::7] = 0.0
    for log in (log_sum, None):
        loss, gradient = ops().distill_loss(x, ids, values, log_sum=log, weight=weight, temperature=1.5)
        alone, _ = ops().distill_loss(x, ids, values, log_sum=log, weight=weight, temperature=1.5, gradient=False)
        assert torch.allclose(alone, loss, rtol=1e-4, atol=1e-5)
        for at in (0, 128, rows - 60):
            part = slice(at, at + 60)
            one, its = ops().distill_loss(x[part], ids[part], values[part], log_sum=None if log is None else log[part], weight=weight[part], temperature=1.5)
            assert torch.allclose(one, loss[part], rtol=1e-4, atol=1e-5)
            assert torch.allclose(its.float(), gradient[part].float(), rtol=1e-4 if dtype == F32 else 2.0**-7, atol=1e-7)


@pytest.mark.parametrize("around", [math.inf, -math.inf, math.nan, 1e30, -1e30])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [37, 3003, 9001, 50257, 131079])
def test_logit_rows_do_not_depend_on_what_lies_around_them(around, dtype, vocab):
    values = random_logits(3, vocab, vocab).to(dtype)
    buf = torch.full((3, vocab + 37), around, dtype=dtype, device=DEV)
    x = buf[:, 5: 5 + vocab]
    x.copy_(values)
    alone = values.to(DEV)
    a, b = ops().top_logits(x, 20, temperature=2.0), ops().top_logits(alone, 20, temperature=2.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.allclose(a[2], b[2], rtol=0, atol=1e-5)
    for log_sum in (None, b[2] + 0.25):
        for gradient in (True, False):
            loss, g = ops().distill_loss(x, b[1], b[0] * 0.5, log_sum=log_sum, temperature=2.0, gradient=gradient)
            want, w = ops().distill_loss(alone, b[1], b[0] * 0.5, log_sum=log_sum, temperature=2.0, gradient=gradient)
            assert torch.allclose(loss, want, rtol=1e-4, atol=1e-5)
            if gradient:
                assert torch.allclose(g.float(), w.float(), rtol=1e-4 if dtype == F32 else 2.0**-7, atol=1e-7)
    arguments = dict(history=i32([[1, 2, 3]] * 3), lengths=i32([3, 2, 1]), presence=f32([1.0] * 3))
    assert torch.equal(ops().adjust_logits(x, **arguments), ops().adjust_logits(alone, **arguments))


# ---- calls in one step, and through the checks --------------------------------------------------

class Other(torch.Tensor):
    pass


def adjusting(rows: int) -> dict:
    return dict(history=i32([[3, 5, 5, 8]] * 4), slots=i32([3, 0, 1][:rows]), lengths=i32([4, 2, 0][:rows]), prompt_lengths=i32([1, 0, 0][:rows]),
                repetition=f32([1.3, 1.0, 2.0][:rows]), presence=f32([0.5, 0.25, 0.0][:rows]), frequency=f32([0.1, 0.0, 1.0][:rows]),
                bias_start=i32([0, 2, 2, 3][: rows + 1]), bias_ids=i32([9, 3, 11]), bias_values=f32([1.0, -2.0, -math.inf]),
                mask=i32([[-2] * 40]), mask_rows=i32([0, -1, 0][:rows]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 3), (0, 4000)])
def test_a_call_in_one_step_is_the_call_through_the_checks(dtype, offset, pad):
    """A subclass's call takes the way through the checks, the same tensor's takes one step."""
    o, x = ops(), rows_at(random_logits(3, 1280, 31), dtype, offset, pad)
    other = x.as_subclass(Other)
    face = o._logit_face("top_logits")
    assert face(x, 5, 1.0, o._error_address(x)) is not None and face(other, 5, 1.0, o._error_address(x)) is None
    for a, b in zip(o.top_logits(x, 7, temperature=2), o.top_logits(other, 7, temperature=2)):
        assert torch.equal(a, b) and a.dtype == b.dtype and a.stride() == b.stride()
    values, ids, log_sum = o.top_logits(x, 7)
    for log in (None, log_sum):
        for a, b in zip(o.distill_loss(x, ids, values, log_sum=log, weight=f32([1.0, 0.0, 0.5])),
                        o.distill_loss(other, ids, values, log_sum=log, weight=f32([1.0, 0.0, 0.5]))):
            assert torch.equal(a, b) and a.stride() == b.stride() and a.data_ptr() % 16 == b.data_ptr() % 16
    assert o.distill_loss(x, ids, values, gradient=False)[1] is None
    a, b = o.adjust_logits(x, **adjusting(3)), o.adjust_logits(other, **adjusting(3))
    assert torch.equal(a, b) and a.stride() == b.stride() and a.data_ptr() % 16 == b.data_ptr() % 16
    whole = x.clone()
    assert o.adjust_logits(whole, **adjusting(3), out=whole) is whole and torch.equal(whole, a)
    one = adjusting(1)
    assert torch.equal(o.adjust_logits(x[:1], **one), a[:1])


def test_logits_of_which_nothing_is_asked():
    x = random_logits(3, 40, 9).to(DEV)
    assert ops().adjust_logits(x) is x
    new = ops().adjust_logits(x, mask=i32([[-1, -1]] * 3))
    assert new is not x and new.data_ptr() != x.data_ptr() and torch.equal(new, x)
    to = torch.empty_like(x)
    assert ops().adjust_logits(x, out=to) is to and torch.equal(to, x)


def test_what_one_step_does_not_take():
    o, x = ops(), random_logits(3, 1280, 5).to(DEV)
    values, ids, log_sum = o.top_logits(x, 7)
    at = o._error_address(x)
    top, adjust, distill = (o._logit_face(name) for name in ("top_logits", "adjust_logits", "distill"))
    for refused in ((x.double(), 5, 1.0, at), (x.cpu(), 5, 1.0, at), (x[0], 5, 1.0, at), (x.t(), 5, 1.0, at), (x[:0], 5, 1.0, at), (x, 0, 1.0, at),
                    (x, 257, 1.0, at), (x, 5.0, 1.0, at), (x, 1 << 70, 1.0, at), (x, 5, 0.0, at), (x, 5, math.nan, at), (x, 5, math.inf, at),
                    (x, 5, "1", at), (x, 5, 1.0), ("x", 5, 1.0, at)):
        assert top(*refused) is None
    good = [x, ids, values, log_sum, 1.0, None, True, None, at]
    assert distill(*good) is not None
    for i, wrong in ((1, ids.long()), (1, ids[:2]), (1, None), (2, values.bfloat16()), (2, values[:, :3]), (3, log_sum[:2]), (3, log_sum.double()),
                     (4, -1.0), (5, log_sum[:1]), (6, 1), (7, x.bfloat16()), (7, x[:, 1:]), (7, ids)):
        assert distill(*good[:i], wrong, *good[i + 1:]) is None, (i, wrong)
    shared = torch.zeros(4 * 1280, device=DEV)
    a, b = shared[: 3 * 1280].view(3, 1280), shared[1280:].view(3, 1280)
    assert distill(a, ids, values, log_sum, 1.0, None, True, b, at) is None
    order = ("history", "slots", "lengths", "prompt_lengths", "repetition", "presence", "frequency", "bias_start", "bias_ids", "bias_values", "mask",
             "mask_rows", "out")
    given = {**dict.fromkeys(order), **adjusting(3)}
    assert adjust(x, *given.values()) is not None
    for name, wrong in (("history", None), ("history", given["history"][0]), ("history", given["history"].long()), ("lengths", None),
                        ("lengths", given["lengths"][:2]), ("slots", given["slots"].float()), ("repetition", given["repetition"].double()),
                        ("bias_start", given["bias_start"][:3]), ("bias_start", None), ("bias_ids", None), ("bias_values", given["bias_values"][:2]),
                        ("mask", given["mask"][:, :39]), ("mask_rows", None), ("out", x[:, :1279]), ("out", x.cpu())):
        assert adjust(x, *{**given, name: wrong}.values()) is None, name


# ---- waits that run out --------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab", [(1, 1031), (3, 50257), (700, 30011)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_waits_that_run_out_leave_nan_and_a_code(rows, vocab, dtype):
    """Every wait for a row's share or for the cluster's sums gives up at once, with copies and sums under way: rows that weigh something are
    NaN, the others 0, the code says so, nothing is written beside the rows, and the next call is right."""
    from research_2_b200.csrc.build import kernel_library

    o = ops()
    case = Distill(rows, vocab, 9, rows, dtype, True, 1.5, 1, 2)
    case.weight[::3] = 0.0
    if rows == 1:
        case.weight[0] = 1.0
    want = case.run()
    entry = kernel_library("distill", {"R2_SHARE_POLLS": 0}).r2_distill
    entry.argtypes = o._LOGIT_SIGNATURES["distill"]
    ids, values, log_sum, weight = (t.to(DEV) for t in (case.ids, case.values, case.log_sum, case.weight))
    loss = torch.full((rows,), -1.0, device=DEV)
    buf = torch.full((rows, vocab + 3), -1.0, dtype=dtype, device=DEV)
    grad = buf[:, 1: 1 + vocab]
    assert entry(0 if dtype == F32 else 1, case.x.data_ptr(), case.x.stride(0), rows, vocab, ids.data_ptr(), values.data_ptr(), 9, log_sum.data_ptr(),
                 weight.data_ptr(), 1.5, loss.data_ptr(), grad.data_ptr(), grad.stride(0), o._error_address(case.x), o._current_stream(0)) == 0
    with pytest.raises(o.KernelTimeout):
        o.raise_on_device_error(DEV)
    weighs = weight != 0
    assert torch.isnan(loss[weighs]).all() and torch.all(loss[~weighs] == 0)
    assert torch.isnan(grad[weighs]).all() and torch.all(grad[~weighs] == 0)
    assert torch.all(buf[:, 0] == -1) and torch.all(buf[:, 1 + vocab:] == -1)
    again = case.run()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    assert o.device_errors(DEV) == 0
