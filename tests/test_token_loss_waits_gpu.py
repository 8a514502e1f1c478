"""Waits that run out in the losses of tokens and their gradients: a build whose warps give up the first sum (of results, having it, or of products, so that those of results wait in vain, 65 ms) marks
everything that depends on it with NaN, leaves its code in the error word and ends; calls behind it are right again."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from tests.test_token_loss_gpu import BF16, DEV, F32, Case, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gives_up", [1, 2])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width,vocab", [(40, 64, 1000), (300, 64, 1000), (300, 1600, 700), (60, 600, 900), (2000, 300, 20000)])
def test_a_wait_that_runs_out_is_marked(rows, width, vocab, dtype, gives_up, monkeypatch):
    from research_2_b200.csrc.build import kernel_library

    o, c = ops(), Case(rows, width, vocab, dtype, rows)
    want = c.run()
    library = kernel_library("token_loss", {"R2_LOSS_GIVES_UP": gives_up})

    def entry(name):
        fn = getattr(library, "r2_" + name)
        fn.argtypes = o._LOGIT_SIGNATURES[name]
        fn.restype = C.c_longlong if name.endswith("_space") else C.c_int
        return fn

    hidden, table = c.hidden.contiguous(), c.table.contiguous()
    code = 0 if dtype == F32 else 1
    size = max(entry("token_loss_space")(code, table.data_ptr(), width, rows, width, vocab, gradient, gradient) for gradient in (0, 1))
    space = torch.empty(size, dtype=torch.uint8, device=DEV)
    loss, log_sum, d_hidden, d_table = (torch.full_like(t, -1.0) for t in want)
    error, stream = o._error_address(hidden), o._current_stream(0)
    assert entry("token_loss")(code, hidden.data_ptr(), width, table.data_ptr(), width, rows, width, vocab, c.targets.data_ptr(), c.weight.data_ptr(), 0.0, 0, loss.data_ptr(),
                               log_sum.data_ptr(), space.data_ptr(), error, stream) == 0
    with pytest.raises(o.KernelTimeout):
        o.raise_on_device_error(DEV)
    assert entry("token_loss_gradient")(code, hidden.data_ptr(), width, table.data_ptr(), width, rows, width, vocab, c.targets.data_ptr(), c.weight.data_ptr(), want[1].data_ptr(), 0.0,
                                        d_hidden.data_ptr(), width, d_table.data_ptr(), width, space.data_ptr(), error, stream) == 0
    with pytest.raises(o.KernelTimeout):
        o.raise_on_device_error(DEV)
    counts = (c.targets >= 0) & (c.targets < vocab) & (c.weight != 0)
    assert torch.isnan(log_sum).all() and torch.isnan(loss[counts]).all() and torch.all(loss[~counts] == 0)
    assert torch.isnan(d_hidden[counts]).all() and torch.all(d_hidden[~counts] == 0)
    assert torch.isnan(d_table).all()
    assert all(torch.equal(a, b) for a, b in zip(c.run(), want))
    assert o.device_errors(DEV) == 0
