"""Arguments that the two ends of a token table refuse on the host, before they look for a device: with tensors of the CPU, so that nothing can be launched."""

import pytest
import torch

from research_2_b200.kernels import ops

X, W, Y, S = torch.zeros(4, 16), torch.zeros(10, 16), torch.zeros(4, dtype=torch.int32), torch.zeros(4)


@pytest.mark.parametrize("call,name", [
    (lambda: ops.token_loss(X, W, None), "targets"), (lambda: ops.token_loss_gradient(X, W, None, S), "targets"), (lambda: ops.token_loss(X[:0], W, None), "targets"),
    (lambda: ops.token_rows(None, W), "ids"), (lambda: ops.token_rows_gradient(None, X, 10), "ids"), (lambda: ops.token_rows_gradient(None, X, 10, into=W), "ids")])
def test_tokens_that_are_not_there(call, name):
    """None is no address: a kernel would read its tokens from 0."""
    with pytest.raises(ops.KernelError, match=name):
        call()


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.4028236e38, float("inf"), float("nan")])
def test_a_scale_that_the_kernel_would_have_as_infinity(scale):
    for call in (lambda: ops.token_rows(Y, W, scale=scale), lambda: ops.token_rows_gradient(Y, X, 10, scale=scale), lambda: ops.token_rows_gradient(Y, X, 10, scale=scale, into=W)):
        with pytest.raises(ops.KernelError, match="scale must be finite"):
            call()
    assert ops._scale(3.4028234663852886e38, "token_rows") == 3.4028234663852886e38
