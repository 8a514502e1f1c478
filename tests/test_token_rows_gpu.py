"""Rows of a table by tokens and the table's gradient, against 64 bits: a row's error is a unit per addition and the rounding of its result."""

from __future__ import annotations

import pytest
import torch

from tests.plain.vocabulary_plain import half_step, rows_gradient
from tests.test_token_loss_gpu import BF16, DEV, F32, gen, ops, strided

pytestmark = pytest.mark.gpu


def tokens(n, vocab, seed, heavy=0.2, outside=True):
    g = gen(seed)
    ids = (vocab * torch.rand(n, generator=g, device=DEV) ** 3).long().clamp_(max=vocab - 1)
    ids = torch.where(torch.rand(n, generator=g, device=DEV) < heavy, vocab // 2, ids)
    if outside and n > 5:
        ids[[1, 3, 5]] = torch.tensor([-1, vocab, 2**31 - 1], device=DEV)
    if n > 6:
        ids[4], ids[6] = 0, vocab - 1
    return ids.to(torch.int32)


def check(ids, above, vocab, scale=1.0, out_dtype=None, into=None):
    want, off = rows_gradient(ids, above, vocab, scale, into)
    before = None if into is None else into.clone()
    got = ops().token_rows_gradient(ids, above, vocab, scale=scale, out_dtype=out_dtype, into=into)
    assert got.dtype == (out_dtype or above.dtype if into is None else into.dtype) and got.shape == (vocab, above.shape[1])
    assert torch.all((got.double() - want).abs() <= off + half_step(got.dtype) * want.abs())
    absent = torch.ones(vocab, dtype=torch.bool, device=DEV)
    absent[ids[(ids >= 0) & (ids < vocab)].long()] = False
    assert torch.equal(got[absent], before[absent]) if into is not None else not got[absent].any()
    return got


SIZES = [(1, 1, 1), (1, 768, 50257), (2, 5, 3), (16, 100, 1031), (31, 33, 7), (64, 64, 64), (100, 257, 300), (1000, 96, 5000), (1024, 768, 50257),
         (2049, 40, 100), (4097, 1600, 3000), (5000, 12, 1), (20000, 64, 128001), (70001, 24, 1000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,width,vocab", SIZES)
def test_gradient(n, width, vocab, dtype):
    above = torch.randn(n, width, generator=gen(n + width), device=DEV).to(dtype)
    check(tokens(n, vocab, n), above, vocab, scale=1.0 if n % 2 else 27.7)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (0, 3), (8, 8), (3, 2)])
def test_types_and_strides(dtype, out_dtype, offset, pad):
    for width in (96, 97):
        above = strided(torch.randn(700, width, generator=gen(3), device=DEV), dtype, offset, pad)
        check(tokens(700, 900, 4), above, 900, out_dtype=out_dtype)
        into = strided(torch.randn(900, width, generator=gen(5), device=DEV), out_dtype, pad, offset)
        check(tokens(700, 900, 6), above, 900, scale=0.5, into=into)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 32, 33, 63, 64, 65, 129, 1000, 4096, 9000])
def test_one_token_alone(n, dtype):
    above = torch.randn(n, 72, generator=gen(n), device=DEV).to(dtype)
    for token in (0, 3, 6):
        check(torch.full((n,), token, dtype=torch.int32, device=DEV), above, 7)


@pytest.mark.parametrize("run", [2, 31, 32, 33, 64, 100])
def test_runs_of_one_length(run):
    ids = torch.arange(50, device=DEV, dtype=torch.int32).repeat_interleave(run)
    ids = ids[torch.randperm(len(ids), generator=gen(run), device=DEV)]
    check(ids, torch.randn(len(ids), 130, generator=gen(1), device=DEV), 61)


def test_order_is_the_places():
    # 2^24 + 1 is no float: what comes first shows
    big, one = 2.0**24, 1.0
    above = torch.tensor([[big], [one], [one], [-big]], device=DEV)
    ids = torch.zeros(4, dtype=torch.int32, device=DEV)
    assert ops().token_rows_gradient(ids, above, 2).tolist() == [[0.0], [0.0]]
    assert ops().token_rows_gradient(ids, above[[1, 2, 0, 3]], 2).tolist() == [[2.0], [0.0]]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_bits_every_time(dtype):
    ids, above = tokens(30000, 2000, 8), torch.randn(30000, 200, generator=gen(9), device=DEV).to(dtype)
    first = ops().token_rows_gradient(ids, above, 2000)
    for _ in range(4):
        assert torch.equal(first, ops().token_rows_gradient(ids, above, 2000))


def test_no_token():
    above = torch.full((300, 40), float("nan"), device=DEV)
    for ids in (torch.full((300,), -1, dtype=torch.int32, device=DEV), torch.full((300,), 50, dtype=torch.int32, device=DEV)):
        assert not ops().token_rows_gradient(ids, above, 50).any()
        into = torch.randn(50, 40, generator=gen(1), device=DEV)
        before = into.clone()
        assert torch.equal(ops().token_rows_gradient(ids, above, 50, into=into), before)
    assert not ops().token_rows_gradient(ids[:0], above[:0], 50).any()
    assert ops().token_rows_gradient(ids, above[:, :0], 50).shape == (50, 0)


def test_nan_stays_with_its_token():
    ids, above = tokens(3000, 200, 10), torch.randn(3000, 64, generator=gen(11), device=DEV)
    clean = ops().token_rows_gradient(ids, above, 200)
    above[7], above[5] = float("nan"), float("inf")    # (place 5 has no token)
    got = ops().token_rows_gradient(ids, above, 200)
    bad = ids[7].item()
    keep = torch.arange(200, device=DEV) != bad
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[bad]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_far_into_a_buffer(dtype):
    # rows from above and table rows beyond 2^31 numbers of their buffers' starts
    above = torch.empty(60_000, 40_000, dtype=dtype, device=DEV)[:, 8:24]
    above.copy_(torch.randn(60_000, 16, generator=gen(12), device=DEV))
    into = torch.empty(60_000, 40_000, dtype=dtype, device=DEV)[:, :16]
    into.zero_()
    check(torch.randint(0, 60_000, (60_000,), generator=gen(13), device=DEV, dtype=torch.int32), above, 60_000, into=into)


def test_broadcast_rows_from_above():
    above = torch.randn(1, 48, generator=gen(14), device=DEV).expand(500, 48)
    check(tokens(500, 60, 15), above, 60)


def test_streams_and_graphs():
    ids, above = tokens(5000, 700, 16), torch.randn(5000, 128, generator=gen(17), device=DEV)
    want = ops().token_rows_gradient(ids, above, 700)
    torch.cuda.synchronize()
    side, late = torch.cuda.Stream(), torch.zeros_like(above)
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        late.copy_(above)
        got = ops().token_rows_gradient(ids, late, 700)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for n in (5000, 3000):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops().token_rows_gradient(ids[:n], above[:n], 700)
        graphs.append((n, graph, out))
    for turn in range(3):
        above.neg_()
        ids.copy_(ids[torch.randperm(5000, generator=gen(turn), device=DEV)])
        torch.cuda.synchronize()
        graphs[0][1].replay()
        with torch.cuda.stream(side):
            graphs[1][1].replay()
        torch.cuda.synchronize()
        for n, _, out in graphs:
            assert torch.equal(out, ops().token_rows_gradient(ids[:n], above[:n], 700))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("out_dtype", [F32, BF16, None])
@pytest.mark.parametrize("n,width,offset,pad", [(1, 1, 0, 0), (50, 100, 0, 0), (300, 768, 8, 8), (77, 33, 3, 2)])
def test_rows(n, width, offset, pad, dtype, out_dtype):
    table = strided(torch.randn(500, width, generator=gen(n), device=DEV), dtype, offset, pad)
    ids = tokens(n, 500, n)
    got = ops().token_rows(ids, table, scale=3.3, out_dtype=out_dtype)
    held = (ids >= 0) & (ids < 500)
    want = torch.where(held[:, None], table[ids.clamp(0, 499).long()].float() * 3.3, 0.0).to(out_dtype or dtype)
    assert got.dtype == want.dtype and torch.equal(got, want)


def test_rows_with_torch_gradients():
    import research_2_b200 as r2

    for dtype in (F32, BF16):
        table = torch.randn(90, 64, generator=gen(1), device=DEV).to(dtype).requires_grad_()
        ids = tokens(60, 90, 2).view(3, 20).long()
        ids[2, 2] = 2**32 + 1
        rows = r2.token_rows(ids, table, scale=2.0, out_dtype=F32)
        assert rows.shape == (3, 20, 64) and rows.dtype == F32 and not rows[2, 2].any()
        rows.sum().backward()    # (what comes from above is one number, broadcast)
        assert table.grad.dtype == dtype
        counts = torch.bincount(ids[(ids >= 0) & (ids < 90)], minlength=90)
        assert torch.equal(table.grad.float(), (2.0 * counts)[:, None].expand(90, 64).to(dtype).float())


def test_refusals():
    o = ops()
    ids, above, table = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(4, 16, device=DEV), torch.zeros(10, 16, device=DEV)
    for bad in (dict(ids=ids.long()), dict(ids=ids[:3]), dict(ids=ids.cpu()), dict(ids=ids.view(2, 2)), dict(above=above.cpu()), dict(above=above.half()),
                dict(above=above[0]), dict(above=above.t().contiguous().t()), dict(vocab=0), dict(vocab=2.5), dict(vocab=2**31), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(into=table[:9]), dict(into=table[:, :8]), dict(into=table.half()), dict(into=table.cpu()),
                dict(into=table[:1].expand(10, 16)), dict(into=table, out_dtype=BF16), dict(out_dtype=torch.float16),
                dict(ids=torch.zeros(6, dtype=torch.int32, device=DEV))):
        call = dict(ids=ids, above=above, vocab=10)
        call.update(bad)
        args = [call.pop(n) for n in ("ids", "above", "vocab")]
        with pytest.raises(o.KernelError):
            o.token_rows_gradient(*args, **call)
    for bad in (dict(ids=ids.long()), dict(ids=ids.view(2, 2)), dict(table=table.cpu()), dict(table=table.half()), dict(table=table[0]),
                dict(table=table.t().contiguous().t()), dict(scale=float("nan")), dict(out_dtype=torch.float16)):
        call = dict(ids=ids, table=table)
        call.update(bad)
        args = [call.pop(n) for n in ("ids", "table")]
        with pytest.raises(o.KernelError):
            o.token_rows(*args, **call)


# tables beyond what gets its zeros beside the sorting (32 MB and some for each token), with rows at and off 16 bytes
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,width,vocab", [(1, 768, 50257), (60, 513, 60001), (1000, 301, 130003), (9, 128, 260000), (33, 127, 400000)])
@pytest.mark.parametrize("tokens", ["any", "ends", "runs", "none"])
def test_tables_whose_zeros_are_written_beside_the_sums(n, width, vocab, dtype, tokens):
    g = torch.Generator(device=DEV).manual_seed(n + width)
    ids = torch.randint(0, vocab, (n,), generator=g, device=DEV, dtype=torch.int32)
    if tokens == "ends":
        ids[: n // 2], ids[n // 2:] = vocab - 1, vocab - 2
        ids[: n // 3] = 0
    elif tokens == "runs":
        ids = vocab - 1 - torch.arange(n, device=DEV, dtype=torch.int32) // 2
    elif tokens == "none":
        ids.fill_(-1)
    above = torch.randn(n, width, generator=g, device=DEV).to(dtype)
    junk = torch.full((vocab * width + 64,), 3.0, dtype=dtype, device=DEV)   # (what the allocator hands out next is not zero)
    del junk
    got = ops().token_rows_gradient(ids, above, vocab)
    want, off = rows_gradient(ids, above, vocab)
    off = off + want.abs() * (torch.finfo(dtype).eps / 2)
    assert torch.all((got.double() - want).abs() <= off)
    assert torch.equal(got, ops().token_rows_gradient(ids, above, vocab))


@pytest.mark.parametrize("n,vocab,which", [(40000, 300, (7,)), (100000, 300, (7, 7 + 148, 299)), (66000, 50257, (13,)), (3000, 2000003, (5, 1999999))])
def test_tokens_that_a_sorting_warp_cannot_list(n, vocab, which):
    """A few tokens at most places: more of a CTA's own than shared memory lists; and more rows than the SMs' CTAs count."""
    g = gen(n)
    ids = torch.randint(0, vocab, (n,), generator=g, device=DEV, dtype=torch.int32)
    often = torch.tensor(which, dtype=torch.int32, device=DEV)[torch.randint(0, len(which), (n,), generator=g, device=DEV)]
    ids = torch.where(torch.rand(n, generator=g, device=DEV) < 0.95, often, ids)
    check(ids, torch.randn(n, 8, generator=g, device=DEV), vocab)
