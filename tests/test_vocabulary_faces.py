"""The two ends of a token table called in one step (`csrc/faces`): what is left to the checks, and the same bits as through them."""

from __future__ import annotations

import pytest
import torch

from research_2_b200.csrc.build import faces_module
from research_2_b200.kernels import ops

DEV = "cuda:0"


def test_what_is_not_plain_is_left_to_the_checks():
    faces, x, w, ids = faces_module(), torch.zeros(2, 40), torch.zeros(9, 40), torch.zeros(2, dtype=torch.int32)
    assert faces.token_loss(x, w, ids, None, 0.0, 0) is None
    assert faces.token_loss_gradient(x, w, ids, torch.zeros(2), None, 0.0, True, True, 0) is None
    assert faces.token_rows(ids, w, 1.0, None) is None and faces.token_rows_gradient(ids, x, 9, 1.0, None) is None
    assert faces.token_loss() is None and faces.token_loss_gradient(x) is None and faces.token_rows(None) is None and faces.token_rows_gradient() is None


@pytest.fixture
def through_checks(monkeypatch):
    def call(f):
        with monkeypatch.context() as m:
            m.setattr(ops, "_faces_built", ops._NoFaces())
            m.setattr(ops, "_logit_faces", {})
            return f()

    return call


def the_same(a, b):
    for one, other in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,), strict=True):
        assert (one is None) == (other is None)
        if one is not None:
            assert one.dtype == other.dtype and one.stride() == other.stride() and torch.equal(one, other)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width,vocab,pad", [(1, 64, 300, 0), (40, 33, 257, 3), (300, 128, 1000, 8)])
def test_the_same_bits(rows, width, vocab, pad, dtype, through_checks):
    g = torch.Generator(device=DEV).manual_seed(rows)
    hidden = torch.randn(rows, width + pad, device=DEV, generator=g).to(dtype)[:, :width]
    table = torch.randn(vocab, width + pad, device=DEV, generator=g).to(dtype)[:, :width]
    targets = torch.randint(-1, vocab + 1, (rows,), dtype=torch.int32, device=DEV, generator=g)
    weight = torch.randn(rows, device=DEV, generator=g)
    for more in (dict(), dict(weight=weight), dict(softcap=20.0), dict(weight=weight, softcap=3)):
        first = ops.token_loss(hidden, table, targets, **more)
        the_same(first, through_checks(lambda: ops.token_loss(hidden, table, targets, **more)))
        for want in (dict(), dict(hidden_gradient=False), dict(table_gradient=False), dict(hidden_gradient=False, table_gradient=False)):
            f = lambda: ops.token_loss_gradient(hidden, table, targets, first[1], **more, **want)   # noqa: E731
            the_same(f(), through_checks(f))
    for more in (dict(), dict(scale=0.5), dict(scale=2, out_dtype=torch.float32), dict(out_dtype=torch.bfloat16)):
        f = lambda: ops.token_rows(targets, table, **more)   # noqa: E731
        the_same(f(), through_checks(f))
        f = lambda: ops.token_rows_gradient(targets, hidden, vocab, **more)   # noqa: E731
        the_same(f(), through_checks(f))


@pytest.mark.gpu
def test_what_only_the_checks_take(through_checks):
    """A subclass, a row that is read for all, numbers that are not Python's own."""
    import numpy as np

    class Sub(torch.Tensor):
        pass

    g = torch.Generator(device=DEV).manual_seed(1)
    hidden, table = torch.randn(4, 40, device=DEV, generator=g), torch.randn(9, 40, device=DEV, generator=g)
    targets = torch.tensor([0, 8, -1, 3], dtype=torch.int32, device=DEV)
    plain = ops.token_loss(hidden, table, targets, softcap=5.0)
    the_same(tuple(t.as_subclass(torch.Tensor) for t in ops.token_loss(hidden.as_subclass(Sub), table, targets, softcap=5.0)), plain)
    the_same(ops.token_loss(hidden, table, targets, softcap=np.float32(5.0)), plain)
    the_same(ops.token_loss(hidden[:1].expand(4, 40), table, targets), ops.token_loss(hidden[:1].repeat(4, 1), table, targets))
    the_same(ops.token_rows_gradient(targets, hidden, np.int64(9)), ops.token_rows_gradient(targets, hidden, 9))
    the_same(ops.token_rows_gradient(targets, hidden[:1].expand(4, 40), 9), ops.token_rows_gradient(targets, hidden[:1].repeat(4, 1), 9))
    for softcap in ("a", None, -1.0, float("inf"), 1e-7, 1e31):
        with pytest.raises((ops.KernelError, TypeError, ValueError)):
            ops.token_loss(hidden, table, targets, softcap=softcap)


@pytest.mark.gpu
def test_scratch_of_a_call_is_of_its_stream():
    """Calls on two streams at once have scratch of their own."""
    g = torch.Generator(device=DEV).manual_seed(2)
    cases = [(torch.randn(200, 96, device=DEV, generator=g), torch.randn(700, 96, device=DEV, generator=g),
              torch.randint(0, 700, (200,), dtype=torch.int32, device=DEV, generator=g)) for _ in range(2)]
    want = []
    for x, w, y in cases:
        loss, log_sum = ops.token_loss(x, w, y)
        want.append((loss, *ops.token_loss_gradient(x, w, y, log_sum), ops.token_rows_gradient(y, x, 700)))
    streams = [torch.cuda.Stream(DEV) for _ in cases]
    torch.cuda.synchronize(DEV)
    got = [None, None]
    for _ in range(5):
        for i, (x, w, y) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                loss, log_sum = ops.token_loss(x, w, y)
                got[i] = (loss, *ops.token_loss_gradient(x, w, y, log_sum), ops.token_rows_gradient(y, x, 700))
    torch.cuda.synchronize(DEV)
    for a, b in zip(got, want):
        the_same(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 100, 200])
def test_a_chain_of_calls_waits_for_what_it_reads(rows, dtype):
    """Each kernel starts beside the one in front of it: a chain in which every call reads what the last one wrote has the bits of one with waits in between."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    vocab, width = 20000, 256
    for _ in range(10):
        ids = torch.randint(0, vocab, (3000,), device=DEV, dtype=torch.int32, generator=g)
        above, hidden = torch.randn(3000, width, device=DEV, generator=g).to(dtype), torch.randn(rows, width, device=DEV, generator=g).to(dtype)
        targets, weight = torch.randint(0, vocab, (rows,), device=DEV, dtype=torch.int32, generator=g), torch.rand(rows, device=DEV, generator=g)

        def chain(wait):
            def step(t):
                if wait:
                    torch.cuda.synchronize(DEV)
                return t

            step(None)
            table = step(ops.token_rows_gradient(ids, above, vocab))
            scaled = step(ops.scale_rows(hidden, weight + 0.5, in_place=False))
            loss, log_sum = step(ops.token_loss(scaled, table, targets, weight=weight))
            d_hidden, d_table = step(ops.token_loss_gradient(scaled, table, targets, log_sum, weight=weight))
            rows_back = step(ops.token_rows_gradient(targets, d_hidden, vocab))
            return (table, loss, log_sum, d_hidden, d_table, rows_back, *step(ops.token_loss(scaled, d_table, targets)))

        first = chain(False)
        the_same(first, chain(True))
