"""The loss of tokens from hidden rows and its gradients against 64 bits (`tests/plain/vocabulary_plain.py`, where the tolerances are derived): sizes
around tiles, both types, strides and alignments, rows without a target, capped logits, infinities and NaN, streams, graphs, refusals."""

from __future__ import annotations

import math

import pytest
import torch

from tests.plain.vocabulary_plain import Loss

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def ops():
    from research_2_b200.kernels import ops as o

    return o


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def strided(values: torch.Tensor, dtype, offset: int = 0, pad: int = 0) -> torch.Tensor:
    """The values as a view that starts `offset` places into rows of `offset + width + pad`; what lies around them is NaN."""
    r, n = values.shape
    buf = torch.full((r, offset + n + pad), float("nan"), dtype=dtype, device=DEV)
    buf[:, offset: offset + n] = values.to(dtype)
    return buf[:, offset: offset + n]


class Case:
    def __init__(self, rows, width, vocab, dtype, seed=0, offset=0, pad=0, table_offset=0, table_pad=0, softcap=0.0, weighted=True, size=2.0):
        g = gen(seed)
        table = torch.randn(vocab, width, generator=g, device=DEV) * (size / math.sqrt(width))
        self.targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
        hidden = torch.randn(rows, width, generator=g, device=DEV) + 2 * torch.rand(rows, 1, generator=g, device=DEV) * table[self.targets.long()]
        if rows > 2:
            self.targets[0], self.targets[1], self.targets[2] = 0, vocab - 1, -100
        if rows > 6:
            self.targets[4], self.targets[5] = vocab, 2**31 - 1
        self.weight = torch.randn(rows, generator=g, device=DEV) if weighted else None
        if weighted and rows > 3:
            self.weight[3] = 0
        self.hidden, self.table = strided(hidden, dtype, offset, pad), strided(table, dtype, table_offset, table_pad)
        self.softcap = softcap

    def kwargs(self):
        return dict(weight=self.weight, softcap=self.softcap)

    def run(self, **wanted):
        loss, log_sum = ops().token_loss(self.hidden, self.table, self.targets, **self.kwargs())
        return loss, log_sum, *ops().token_loss_gradient(self.hidden, self.table, self.targets, log_sum, **self.kwargs(), **wanted)

    def plain(self):
        return Loss(self.hidden, self.table, self.targets, self.weight, self.softcap)

    def check(self):
        got, want = self.run(), self.plain()
        ops().raise_on_device_error(DEV)
        for name, t in zip(("loss", "log_sum", "d_hidden", "d_table"), got):
            exact, off = getattr(want, name), getattr(want, name + "_off")
            worst = ((t.double() - exact).abs() / off.clamp(min=1e-300)).nan_to_num(nan=math.inf).max().item()
            assert torch.all((t.double() - exact).abs() <= off), (name, worst)
        assert got[0].dtype == got[1].dtype == F32 and got[2].dtype == self.hidden.dtype and got[3].dtype == self.table.dtype
        return got


SIZES = [(1, 64, 300), (1, 768, 50257), (3, 100, 1031), (17, 33, 257), (5, 8, 1), (64, 1, 7), (128, 64, 256), (129, 72, 513), (256, 128, 512),
         (257, 200, 1000), (300, 768, 2049), (1000, 48, 5000), (600, 320, 20011)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width,vocab", SIZES)
def test_against_64_bits(rows, width, vocab, dtype):
    Case(rows, width, vocab, dtype, seed=rows + vocab).check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset,pad,table_offset,table_pad", [(1, 0, 0, 0), (0, 8, 8, 0), (0, 1, 0, 3), (4, 4, 4, 12), (8, 24, 16, 40)])
def test_strides_and_alignments(dtype, offset, pad, table_offset, table_pad):
    Case(140, 96, 700, dtype, 5, offset, pad, table_offset, table_pad).check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("softcap,size", [(30.0, 2.0), (5.0, 6.0), (0.3, 1.0), (1000.0, 2.0)])
def test_capped(dtype, softcap, size):
    Case(200, 128, 900, dtype, 6, softcap=softcap, size=size).check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_weights(dtype):
    Case(70, 64, 500, dtype, 7, weighted=False).check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e-4, 40.0, 300.0])
def test_flat_and_steep_rows(dtype, size):
    Case(65, 128, 777, dtype, 8, size=size).check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_table_beyond_32_bits(dtype):
    # rows 40,000 numbers apart: the last ones lie more than 2^31 numbers into the buffer
    c = Case(20, 64, 100, dtype, 9)
    vocab, ld = 60_000, 40_000
    buffer = torch.empty(vocab, ld, dtype=dtype, device=DEV)
    c.table = buffer[:, :64]
    c.table.copy_(torch.randn(vocab, 64, generator=gen(10), device=DEV) / 4)
    c.targets = torch.randint(0, vocab, (20,), generator=gen(11), device=DEV, dtype=torch.int32)
    c.targets[0] = vocab - 1
    c.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_broadcast_rows(dtype):
    c = Case(9, 64, 300, dtype, 12)
    c.hidden = c.hidden[:1].expand(9, 64)
    c.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_gradient_alone(dtype):
    c = Case(150, 64, 600, dtype, 13)
    _, _, d_hidden, d_table = c.run()
    _, _, only, none = c.run(table_gradient=False)
    assert none is None and torch.equal(only, d_hidden)
    _, _, none, only = c.run(hidden_gradient=False)
    assert none is None and torch.equal(only, d_table)
    assert c.run(hidden_gradient=False, table_gradient=False)[2:] == (None, None)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_bits_every_time(dtype):
    c = Case(500, 320, 9001, dtype, 14)
    first = c.run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, c.run()))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_without_a_target_may_hold_anything(dtype):
    c = Case(300, 64, 700, dtype, 15)
    c.targets[200:] = -1
    c.targets[:200] = c.targets[:200].clamp(0, 699)
    c.weight[:200] = 1.0
    clean = c.run()
    c.hidden[200:] = float("nan")
    c.hidden[250] = float("inf")
    loss, log_sum, d_hidden, d_table = c.run()
    assert torch.equal(loss, clean[0]) and torch.equal(log_sum[:200], clean[1][:200])
    assert torch.equal(d_hidden, clean[2]) and torch.equal(d_table, clean[3])
    assert torch.all(loss[200:] == 0) and torch.all(d_hidden[200:] == 0)
    c.targets[200:], c.weight[200:] = 5, 0.0
    again = c.run()
    assert torch.equal(again[0], loss) and torch.equal(again[2], d_hidden) and torch.equal(again[3], d_table)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_row_counts(dtype):
    c = Case(40, 64, 700, dtype, 16)
    c.targets[:] = -1
    c.hidden[3] = float("nan")
    loss, _, d_hidden, d_table = c.run()
    assert not loss.any() and not d_hidden.any() and not d_table.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinities_and_nan_stay_in_their_row(dtype):
    c = Case(130, 64, 600, dtype, 17)
    c.targets[:] = 7
    clean = ops().token_loss(c.hidden, c.table, c.targets)
    c.hidden[5], c.hidden[9, 3], c.hidden[128] = float("nan"), float("inf"), -float("inf")
    got = ops().token_loss(c.hidden, c.table, c.targets)
    bad = torch.zeros(130, dtype=torch.bool, device=DEV)
    bad[[5, 9, 128]] = True
    for a, b in zip(got, clean):
        assert torch.equal(a[~bad], b[~bad]) and not torch.isfinite(a[bad]).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forbidden_tokens(dtype):
    # a table with rows that make every logit -inf: such tokens have no share, and a row whose target is one has an infinite loss
    c = Case(20, 64, 300, dtype, 18, weighted=False)
    c.hidden[:, 0] = 1.0
    c.table[10:290] = 0.0
    c.table[10:290, 0] = -float("inf")
    c.targets[:] = 3
    c.targets[4] = 100
    loss, log_sum = ops().token_loss(c.hidden, c.table, c.targets)
    keep = [v for v in range(300) if not 10 <= v < 290]
    want = Loss(c.hidden, c.table[keep], torch.full_like(c.targets, 3))
    assert torch.all((log_sum.double() - want.log_sum).abs() <= want.log_sum_off)
    assert loss[4].item() == math.inf and torch.isfinite(loss[torch.arange(20, device=DEV) != 4]).all()


def test_no_rows():
    for dtype in (F32, BF16):
        c = Case(0, 64, 50, dtype)
        c.weight = None
        loss, log_sum, d_hidden, d_table = c.run()
        assert loss.shape == log_sum.shape == (0,) and d_hidden.shape == (0, 64)
        assert d_table.shape == (50, 64) and not d_table.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_against_differences(dtype):
    c = Case(12, 40, 90, dtype, 19, softcap=8.0)
    _, _, d_hidden, d_table = c.run()
    g = gen(20)
    for which, grad in (("hidden", d_hidden), ("table", d_table)):
        base = getattr(c, which).double()
        step = torch.randn(base.shape, generator=g, device=DEV, dtype=torch.float64)
        h = 1e-5

        def total(sign):
            moved = base + sign * h * step
            x, w = (moved, c.table.double()) if which == "hidden" else (c.hidden.double(), moved)
            return Loss(x, w, c.targets, c.weight, 8.0).loss.sum().item()

        want = (total(1) - total(-1)) / (2 * h)
        off = (c.plain().__dict__["d_" + which + "_off"] * step.abs()).sum().item() + 1e-7
        assert abs((grad.double() * step).sum().item() - want) <= off


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_another_stream(dtype):
    c = Case(200, 128, 3000, dtype, 21)
    want = c.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    hidden = torch.zeros_like(c.hidden)
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        hidden.copy_(c.hidden)      # arrives late, on the stream of the call
        c.hidden = hidden
        got = c.run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_and_replayed(dtype):
    cases = [Case(200, 128, 3000, dtype, 22), Case(77, 64, 1500, dtype, 23)]
    wants = [c.run() for c in cases]
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = c.run()
        graphs.append((graph, out))
    # two graphs in turn and side by side: neither has the other's scratch
    side = torch.cuda.Stream()
    for _ in range(3):
        for c in cases:
            c.hidden.neg_()
        torch.cuda.synchronize()
        changed = [c.run() for c in cases]
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, changed):
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    for c in cases:
        c.hidden.neg_()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], wants[0]))


def test_nothing_around_the_results_is_written():
    c = Case(130, 72, 515, BF16, 24, offset=8, pad=8, table_offset=8, table_pad=8)
    before = [t.clone() for t in (c.hidden, c.table, c.targets, c.weight)]
    c.run()
    assert all(torch.equal(a, b) for a, b in zip(before, (c.hidden, c.table, c.targets, c.weight)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_with_torch_gradients(dtype, kind):
    import research_2_b200 as r2

    c = Case(90, 64, 400, dtype, 25, softcap=12.0)
    hidden, table = c.hidden.clone().requires_grad_(), c.table.clone().requires_grad_()
    above = torch.randn(90, generator=gen(26), device=DEV)
    targets = c.targets.to(kind)
    if kind is torch.int64:
        targets[7] = 2**32 + 5    # no token, and none after a cut to 32 bits
    loss = r2.token_loss(hidden, table, targets, weight=c.weight, softcap=12.0)
    (loss * above).sum().backward(retain_graph=True)
    held = torch.where((targets >= 0) & (targets < 400), targets, -1).to(torch.int32)
    want = Loss(c.hidden, c.table, held, c.weight * above, 12.0)
    for got, name in ((hidden.grad, "d_hidden"), (table.grad, "d_table")):
        # (weight * above is rounded to float32: a unit more)
        assert torch.all((got.double() - getattr(want, name)).abs() <= getattr(want, name + "_off") + 2.0**-24 * getattr(want, name).abs())
    first = hidden.grad.clone(), table.grad.clone()
    hidden.grad = table.grad = None
    (loss * above).sum().backward()     # a kept graph, a second time
    assert torch.equal(hidden.grad, first[0]) and torch.equal(table.grad, first[1])
    frozen = r2.token_loss(hidden, table.detach(), targets, weight=c.weight, softcap=12.0)
    assert torch.equal(torch.autograd.grad((frozen * above).sum(), hidden)[0], first[0])
    with pytest.raises(ops().KernelError, match="detach"):
        r2.token_loss(hidden, table, targets, weight=c.weight.clone().requires_grad_())


def test_gradients_of_broadcast_rows():
    import research_2_b200 as r2

    c = Case(6, 64, 200, F32, 27, weighted=False)
    c.targets[:] = torch.arange(6, device=DEV)
    row = c.hidden[:1].clone().requires_grad_()
    r2.token_loss(row.expand(6, 64), c.table, c.targets).sum().backward()
    c.hidden = row.detach().expand(6, 64)
    want = c.plain()
    assert row.grad.shape == (1, 64)
    assert torch.all((row.grad.double() - want.d_hidden.sum(0, keepdim=True)).abs() <= want.d_hidden_off.sum(0, keepdim=True) * 2)


def test_a_tied_table_from_both_ends():
    """Look up, a layer of torch's, the loss over the same table, both gradients, a step; then again."""
    import research_2_b200 as r2

    torch.manual_seed(0)
    vocab, width = 1031, 64
    table = (torch.randn(vocab, width, device=DEV) / 8).requires_grad_()
    mix = (torch.randn(width, width, device=DEV) / 8).requires_grad_()
    ids = torch.randint(0, vocab, (2, 33), device=DEV)
    weight = torch.full((64,), 1.0 / 64, device=DEV)

    def step(table, mix, rows, loss):
        x = rows(ids[:, :-1], table)
        h = torch.tanh(x.reshape(-1, width) @ mix)
        return torch.autograd.grad(loss(h, table), (table, mix))

    plain_rows = lambda i, t: t[i] * 8.0
    plain_loss = lambda h, t: torch.nn.functional.cross_entropy(h @ t.t(), ids[:, 1:].reshape(-1))
    for _ in range(2):
        got = step(table, mix, lambda i, t: r2.token_rows(i, t, scale=8.0), lambda h, t: r2.token_loss(h, t, ids[:, 1:].reshape(-1), weight=weight).sum())
        want = step(table.double().detach().requires_grad_(), mix.double().detach().requires_grad_(), plain_rows, plain_loss)
        for a, b in zip(got, want):
            # (torch's own products in float32 stand between: 64 terms, twice, and a tanh)
            assert (a.double() - b).abs().max().item() <= 1e-4 * b.abs().max().item()
        with torch.no_grad():
            table -= 0.1 * got[0]
            mix -= 0.1 * got[1]
    # the same by the operators alone, one buffer for both ends
    with torch.no_grad():
        rows = ops().token_rows(ids[:, :-1].reshape(-1).to(torch.int32), table, scale=8.0)
        h = torch.tanh(rows @ mix)
        y = ids[:, 1:].reshape(-1).to(torch.int32)
        loss, log_sum = ops().token_loss(h, table, y, weight=weight)
        d_h, d_table = ops().token_loss_gradient(h, table, y, log_sum, weight=weight)
        ops().token_rows_gradient(ids[:, :-1].reshape(-1).to(torch.int32), (d_h * (1 - h * h)) @ mix.t(), vocab, scale=8.0, into=d_table)
    want = step(table.double().detach().requires_grad_(), mix.double().detach().requires_grad_(), plain_rows, plain_loss)[0]
    assert (d_table.double() - want).abs().max().item() <= 1e-4 * want.abs().max().item()


def test_refusals():
    o = ops()
    x, w = torch.zeros(4, 16, device=DEV), torch.zeros(10, 16, device=DEV)
    y, s = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(4, device=DEV)
    for bad in (dict(hidden=x.cpu()), dict(hidden=x[0]), dict(hidden=x.half()), dict(hidden=x.bfloat16()), dict(table=w[:, :8]), dict(table=w.t().contiguous().t()),
                dict(hidden=x.t().contiguous().t()), dict(table=w[:0]), dict(targets=y.long()), dict(targets=y[:3]), dict(targets=y.cpu()),
                dict(targets=torch.zeros(8, dtype=torch.int32, device=DEV)[::2]), dict(weight=s.double()), dict(weight=s[:2]), dict(softcap=-1.0),
                dict(softcap=math.nan), dict(softcap=math.inf), dict(softcap=1e-7), dict(softcap=1e31), dict(hidden=x[:, :0], table=w[:, :0])):
        call = dict(hidden=x, table=w, targets=y, weight=None, softcap=0.0)
        call.update(bad)
        args = [call.pop(n) for n in ("hidden", "table", "targets")]
        with pytest.raises(o.KernelError):
            o.token_loss(*args, **call)
        with pytest.raises(o.KernelError):
            o.token_loss_gradient(*args, s, **call)
    for log_sum in (None, s[:3], s.double(), s.cpu()):
        with pytest.raises(o.KernelError):
            o.token_loss_gradient(x, w, y, log_sum)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_without_a_target_beside_a_table_with_infinities(dtype):
    # products of a left-out row's place and an infinity are nothing
    c = Case(300, 64, 700, dtype, 28)
    c.targets[:] = 3
    c.targets[70:] = -1
    c.weight[:] = 1.0
    c.hidden[:, 0], c.table[:, 0], c.table[500:] = 1.0, 0.0, 0.0
    c.table[500:, 0] = -float("inf")
    loss, log_sum, d_hidden, d_table = c.run()
    keep = Loss(c.hidden, c.table[:500], c.targets, c.weight)
    assert torch.all((loss.double() - keep.loss).abs() <= keep.loss_off)
    assert torch.isfinite(d_table).all() and not d_table[500:].any() and not d_hidden[70:].any()
    assert torch.all((d_table[:500].double() - keep.d_table).abs() <= keep.d_table_off)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [20, 200])
@pytest.mark.parametrize("softcap", [1e4, 1e8, 1e30])
def test_a_cap_far_above_the_logits_changes_nothing(dtype, rows, softcap):
    # |logits| below 40: their cube over 3 cap^2 is below 3e-4; the tanh is off by 2e-6 of itself at most, as much again in the slope
    c = Case(rows, 96, 700, dtype, 29, softcap=softcap)
    got, want = c.run(), Loss(c.hidden, c.table, c.targets, c.weight)
    assert want.z.abs().max().item() < 40
    moved = 40**3 / (3 * softcap**2) + 2e-6 * 40
    a = torch.where((c.targets >= 0) & (c.targets < 700), c.weight, 0.0).double().abs()
    assert torch.all((got[1].double() - want.log_sum).abs() <= want.log_sum_off + moved)
    assert torch.all((got[0].double() - want.loss).abs() <= want.loss_off + 2 * a * moved)
    # a factor moves by its exponent's error and its slope's; the rounding counts again on what moved
    p = torch.exp(want.z - want.log_sum[:, None])
    dz = (2.1 * (2 * moved + 40**2 / softcap**2 + 4e-6)) * a[:, None] * p.scatter_add(1, c.targets.clamp(0, 699).long()[:, None], torch.ones(rows, 1, dtype=p.dtype, device=DEV))
    assert torch.all((got[2].double() - want.d_hidden).abs() <= want.d_hidden_off + dz @ c.table.double().abs())
    assert torch.all((got[3].double() - want.d_table).abs() <= want.d_table_off + dz.t() @ torch.where(a[:, None] != 0, c.hidden.double(), 0.0).abs())


def test_rows_of_any_shape_with_torch_gradients():
    import research_2_b200 as r2

    c = Case(60, 64, 400, F32, 30)
    hidden, table = c.hidden.clone().requires_grad_(), c.table.clone().requires_grad_()
    flat = r2.token_loss(hidden, table, c.targets, weight=c.weight)
    want = torch.autograd.grad(flat.sum(), (hidden, table))
    shaped = r2.token_loss(hidden.view(3, 20, 64), table, c.targets.view(3, 20), weight=c.weight.view(3, 20))
    assert shaped.shape == (3, 20) and torch.equal(shaped.reshape(-1), flat)
    got = torch.autograd.grad(shaped.sum(), (hidden, table))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = hidden.detach().t().contiguous().t().requires_grad_()
    wide = table.detach().t().contiguous().t().requires_grad_()
    got = torch.autograd.grad(r2.token_loss(turned, wide, c.targets, weight=c.weight).sum(), (turned, wide))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for bad in (dict(targets=c.targets[:5]), dict(weight=c.weight[:5]), dict(targets=c.targets.float()), dict(table=table[0])):
        call = dict(table=table, targets=c.targets, weight=None)
        call.update(bad)
        with pytest.raises(ops().KernelError):
            r2.token_loss(hidden, **call)


def test_gradients_captured_into_a_graph():
    import research_2_b200 as r2

    c = Case(150, 64, 900, BF16, 31)
    hidden, table = c.hidden.clone().requires_grad_(), c.table.clone().requires_grad_()

    def step():
        return torch.autograd.grad(r2.token_loss(hidden, table, c.targets, weight=c.weight).sum(), (hidden, table))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        hidden.neg_()
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width,vocab,softcap", [(1, 1600, 1000, 0.0), (20, 1032, 900, 25.0), (128, 2500, 700, 0.0), (300, 1600, 1500, 0.0), (260, 4100, 400, 30.0)])
def test_long_rows(rows, width, vocab, softcap, dtype):
    Case(rows, width, vocab, dtype, 32, softcap=softcap).check()


@pytest.mark.parametrize("rows", [100, 300])
def test_float32_is_no_further_off_than_float32_sums(rows):
    """What rounds towards zero 96 times and more shows as a bias: the logits of one token, 1,536 products each, against 64 bits, beside torch's own
    (whose error is what rounding to nearest leaves)."""
    g = gen(33)
    x, w = torch.randn(rows, 1536, generator=g, device=DEV), torch.randn(1, 1536, generator=g, device=DEV)
    exact = (x.double() @ w.double().t())[:, 0]
    _, log_sum = ops().token_loss(x, w, torch.zeros(rows, dtype=torch.int32, device=DEV))
    size = exact.pow(2).mean().sqrt()
    # six pieces of 256 products: 16 additions of up to a unit each to a part of it, which grows; half of the units' mean, rounding to nearest above
    assert (log_sum.double() - exact).pow(2).mean().sqrt() <= 16 * 2.0**-24 * size


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_table_that_is_read_where_it_lies_is_not_copied(dtype):
    rows, width, vocab = 64, 256, 20000
    c = Case(rows, width, vocab, dtype, 23)
    c.run()

    def extra(call):
        before = torch.cuda.memory_allocated(DEV)
        torch.cuda.reset_peak_memory_stats(DEV)
        out = call()
        peak = torch.cuda.max_memory_allocated(DEV) - before
        return out, peak - sum(t.numel() * t.element_size() for t in out if t is not None)

    table, planes = vocab * width * c.table.element_size(), 1 if dtype is BF16 else 3
    (loss, log_sum), most = extra(lambda: ops().token_loss(c.hidden, c.table, c.targets))
    assert most < table / 4
    # the gradient's factors are bfloat16 [256, vocab] in as many planes, the rows as many of [256, width]
    factors = 256 * (vocab + 256 + width) * 2 * planes
    _, most = extra(lambda: ops().token_loss_gradient(c.hidden, c.table, c.targets, log_sum, hidden_gradient=False))
    assert most < factors + table / 4


@pytest.mark.parametrize("rows,width,vocab", [(3, 768, 2000), (40, 64, 1500), (128, 200, 3000), (300, 96, 2500)])
def test_what_rounding_leaves_of_a_tokens_own_factor_is_added(rows, width, vocab):
    """bfloat16, tokens that the model finds unlikely: a row's factor is nearly all at its own token, a (p - 1). Its rounding, half a step of |a (p - 1)| times the row of the
    other operand, is not in the hidden rows' gradient, and of up to 128 rows not in the table's: the tolerance is the oracle's without it (4 units of 2^-24 in its place)."""
    c = Case(rows, width, vocab, BF16, rows, size=0.05)
    got, want = c.run(), c.plain()
    a = torch.where((c.targets >= 0) & (c.targets < vocab), c.weight.double(), 0.0)
    y = c.targets.clamp(0, vocab - 1).long()
    own = a * torch.expm1(want.z.gather(1, y[:, None])[:, 0] - want.log_sum)
    less = (2.0**-8 - 4 * 2.0**-24) * own.abs()[:, None]
    x, w = torch.where(a[:, None] != 0, c.hidden.double(), 0.0), c.table.double()
    off = want.d_hidden_off - less * w[y].abs()
    assert torch.all((got[2].double() - want.d_hidden).abs() <= off)
    if rows <= 128:
        off = want.d_table_off.index_add(0, y, -less * x.abs())
        assert torch.all((got[3].double() - want.d_table).abs() <= off)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [100, 300])
def test_one_token_for_all_rows(dtype, rows):
    for token in (0, 40, 599):
        c = Case(rows, 96, 600, dtype, 31)
        c.targets[7:] = token
        c.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(20, 700001), (100, 530000), (300, 400003)])
def test_several_pieces_of_the_vocabulary(rows, vocab, dtype):
    """More tokens than a piece of the factors holds: targets in every piece."""
    c = Case(rows, 24, vocab, dtype, 41)
    c.targets[8], c.targets[9], c.targets[10] = vocab - 2, vocab // 2, 524288 if vocab > 524288 else 262144
    c.check()


@pytest.mark.parametrize("rows,width,vocab", [(1, 768, 20011), (16, 300, 30000), (17, 257, 40001), (33, 1031, 25000), (64, 96, 70000), (40, 24, 530001)])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_few_float32_rows_at_large_tables(rows, width, vocab, softcap):
    """Tables of more tiles than the GPU holds at once: the loss reads them as they are, the hidden rows' gradient their planes."""
    pad = -width % 4
    c = Case(rows, width, vocab, F32, rows, table_pad=pad, softcap=softcap)
    c.check()
    again = c.run()
    assert all(torch.equal(a, b) for a, b in zip(again, c.run()))


@pytest.mark.parametrize("rows,vocab", [(20, 1100003), (100, 1048833), (300, 600001)])
def test_several_pieces_of_a_bfloat16_vocabulary(rows, vocab):
    """Targets at both sides of where pieces end, first and last tokens; few rows with what rounding leaves in every piece."""
    c = Case(rows, 16, vocab, BF16, 43)
    c.targets[7:14] = torch.tensor([524287, 524288, vocab - 2, vocab // 2, 262143, 524032, vocab - 257], dtype=torch.int32, device=DEV)
    c.check()
