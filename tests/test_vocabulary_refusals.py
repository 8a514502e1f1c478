"""Sizes that the two ends of a token table refuse before they look for a device."""

import pytest
import torch

from research_2_b200.kernels import ops


def test_sizes_whose_indexes_pass_32_bits():
    many, one, tokens = torch.empty(1, 1).expand(2**30 + 1, 1), torch.empty(1, 1), torch.zeros(1, dtype=torch.int32)
    wide = torch.empty(1).expand(1, 2**32 + 1)
    for call in (lambda: ops.token_loss(many, one, tokens), lambda: ops.token_loss_gradient(many, one, tokens, None), lambda: ops.token_loss(wide, wide, tokens),
                 lambda: ops.token_rows(tokens, many), lambda: ops.token_rows(tokens, wide), lambda: ops.token_rows_gradient(tokens, many, 10),
                 lambda: ops.token_rows_gradient(tokens, wide, 10)):
        with pytest.raises(ops.KernelError, match="2\\^30"):
            call()
