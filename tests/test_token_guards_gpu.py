"""What lies around the results of the two ends of a token table stays as it was, bit for bit: losses, gradients and scratch between guards, rows of results further apart than they are wide, results off 16 bytes."""

from __future__ import annotations

import pytest
import torch

from tests.test_token_loss_gpu import BF16, DEV, F32, Case, gen, ops

pytestmark = pytest.mark.gpu
GUARD = 0x5A


class Guarded:
    """A matrix (or a vector) of `rows` rows `ld` numbers apart, `offset` numbers into a buffer of guard bytes, 4 KB of them behind it."""

    def __init__(self, rows, width, ld, offset, dtype):
        size = torch.empty(0, dtype=dtype).element_size()
        self.bytes = torch.full((offset * size + rows * ld * size + 4096,), GUARD, dtype=torch.uint8, device=DEV)
        self.t = self.bytes[offset * size: (offset + rows * ld) * size].view(dtype).view(rows, ld)[:, :width]
        self.ld = ld
        self.inside = torch.zeros_like(self.bytes, dtype=torch.bool)
        self.inside[offset * size: (offset + rows * ld) * size].view(rows, ld * size)[:, : width * size] = True

    def check(self, want):
        assert torch.equal(self.t, want)
        assert torch.all(self.bytes[~self.inside] == GUARD)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 0), (0, 1), (5, 3), (16, 8)])
@pytest.mark.parametrize("rows,width,vocab,softcap", [(5, 33, 257, 0.0), (127, 72, 515, 9.0), (129, 100, 1031, 0.0), (300, 264, 771, 0.0), (513, 65, 260, 0.0)])
def test_losses(rows, width, vocab, softcap, pad, offset, dtype):
    o, c = ops(), Case(rows, width, vocab, dtype, rows, softcap=softcap)
    want = c.run()
    hidden, table = c.hidden.contiguous(), c.table.contiguous()
    code, space_of = 0 if dtype == F32 else 1, o._logit_entry("token_loss_space")
    error, stream = o._error_address(hidden), o._current_stream(0)
    loss, log_sum = Guarded(1, rows, rows, offset, F32), Guarded(1, rows, rows, offset, F32)
    space = Guarded(1, *(space_of(code, table.data_ptr(), width, rows, width, vocab, 0, 0),) * 2, 0, torch.uint8)
    assert o._logit_entry("token_loss")(code, hidden.data_ptr(), width, table.data_ptr(), width, rows, width, vocab, c.targets.data_ptr(), c.weight.data_ptr(), softcap, 0,
                                        loss.t.data_ptr(), log_sum.t.data_ptr(), space.t.data_ptr(), error, stream) == 0
    loss.check(want[0][None])
    log_sum.check(want[1][None])
    assert torch.all(space.bytes[~space.inside] == GUARD)
    for both in (True, False):
        d_hidden, d_table = Guarded(rows, width, width + pad, offset, dtype), Guarded(vocab, width, width + pad, offset, dtype)
        space = Guarded(1, *(space_of(code, table.data_ptr(), width, rows, width, vocab, 1, int(both)),) * 2, 0, torch.uint8)
        assert o._logit_entry("token_loss_gradient")(
            code, hidden.data_ptr(), width, table.data_ptr(), width, rows, width, vocab, c.targets.data_ptr(), c.weight.data_ptr(), want[1].data_ptr(), softcap,
            d_hidden.t.data_ptr() if both else 0, d_hidden.ld, d_table.t.data_ptr(), d_table.ld, space.t.data_ptr(), error, stream) == 0
        if both:
            d_hidden.check(want[2])
        d_table.check(want[3])
        assert torch.all(space.bytes[~space.inside] == GUARD)
    assert o.device_errors(DEV) == 0


@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("tokens,width,vocab,pad,offset", [(1, 1, 1, 0, 1), (7, 33, 30, 3, 1), (300, 264, 1031, 8, 0), (1000, 96, 50, 5, 8), (3000, 40, 100003, 0, 0), (2, 1024, 20000, 0, 0)])
def test_rows(tokens, width, vocab, pad, offset, dtype, out_dtype):
    o, g = ops(), gen(tokens)
    ids = torch.randint(-1, vocab + 1, (tokens,), generator=g, device=DEV, dtype=torch.int32)
    table, above = torch.randn(vocab, width, generator=g, device=DEV).to(dtype), torch.randn(tokens, width, generator=g, device=DEV).to(dtype)
    code, out_code, stream = (0 if dtype == F32 else 1), (0 if out_dtype == F32 else 1), o._current_stream(0)
    rows = Guarded(tokens, width, width + pad, offset, out_dtype)
    assert o._logit_entry("token_rows")(code, out_code, ids.data_ptr(), table.data_ptr(), width, rows.t.data_ptr(), rows.ld, tokens, width, vocab, 1.5, stream) == 0
    rows.check(o.token_rows(ids, table, scale=1.5, out_dtype=out_dtype))
    size = o._logit_entry("token_rows_space")(tokens, width, vocab)
    base = torch.randn(vocab, width, generator=g, device=DEV).to(out_dtype)
    for add in (1, 0) if pad == 0 and offset == 0 else (1,):   # (a new table is one piece at 16 bytes)
        out, space = Guarded(vocab, width, width + pad, offset, out_dtype), Guarded(1, size, size, 0, torch.uint8)
        out.t.copy_(base)
        assert o._logit_entry("token_rows_gradient")(code, out_code, ids.data_ptr(), above.data_ptr(), width, out.t.data_ptr(), out.ld, tokens, width, vocab, 0.5, add, space.t.data_ptr(), stream) == 0
        out.check(o.token_rows_gradient(ids, above, vocab, scale=0.5, into=base.clone()) if add else o.token_rows_gradient(ids, above, vocab, scale=0.5, out_dtype=out_dtype))
        assert torch.all(space.bytes[~space.inside] == GUARD)
