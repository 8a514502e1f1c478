"""Edges of the two ends of a token table for autograd: rows of no numbers, a table of no tokens."""

import pytest
import torch

import research_2_b200 as r2
from research_2_b200.kernels import ops


@pytest.mark.parametrize("shape", [(3,), (2, 3), (0,)])
def test_hidden_rows_of_no_numbers_are_refused(shape):
    with pytest.raises(ops.KernelError, match="numbers"):
        r2.token_loss(torch.zeros(*shape, 0), torch.zeros(5, 0), torch.zeros(shape, dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_a_table_of_no_tokens(dtype):
    table = torch.zeros(0, 8, device="cuda", dtype=dtype, requires_grad=True)
    rows = r2.token_rows(torch.tensor([[0, 3, -1]], device="cuda"), table)
    assert rows.shape == (1, 3, 8) and not rows.any()
    rows.sum().backward()
    assert table.grad.shape == (0, 8) and table.grad.dtype == dtype
