"""Where the faces cannot be built, operators on rows of logits are called through ctypes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from research_2_b200.csrc.build import BuildError
from research_2_b200.kernels import ops


@pytest.fixture
def no_faces(monkeypatch):
    tries = []

    def faces_module():
        tries.append(1)
        raise BuildError("no Python.h")

    monkeypatch.setattr(ops, "faces_module", faces_module)
    monkeypatch.setattr(ops, "_faces_built", None, raising=False)
    monkeypatch.setattr(ops, "_logit_faces", {})
    return tries


def test_faces_that_cannot_be_built_are_said_once(no_faces, monkeypatch):
    monkeypatch.setattr(ops, "_logit_entry", lambda name: ops.C.CFUNCTYPE(ops.C.c_int)(lambda: 0))
    monkeypatch.setattr(ops, "_libs", {"top_logits": object(), "distill": object()})
    with pytest.warns(UserWarning, match="Python.h"):
        assert ops._logit_face("top_logits")(torch.zeros(2, 4), 1, 1.0, 0) is None
    assert ops._logit_face("distill")() is None and ops._logit_face("top_logits")() is None
    assert len(no_faces) == 1


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:operators on rows of logits")
def test_operators_without_faces(no_faces):
    x = torch.randn(3, 1031, device="cuda:0")
    values, ids, log_sum = ops.top_logits(x, 5)
    assert torch.equal(values, torch.topk(x, 5, dim=1).values)
    loss, gradient = ops.distill_loss(x, ids, values, log_sum=log_sum)
    assert torch.all(loss.abs() < 1e-5) and torch.all(gradient.abs() < 1e-5)   # a student that is its teacher
    assert torch.equal(ops.adjust_logits(x, mask=torch.full((3, 33), -1, dtype=torch.int32, device="cuda:0")), x)
    assert len(no_faces) == 1


@pytest.mark.gpu
def test_numbers_that_are_not_python_s_own():
    """The face takes Python's numbers; the checks behind it whatever is one."""
    x = torch.randn(3, 1031, device="cuda:0")
    want = ops.top_logits(x, 5, temperature=2.0)
    for k, temperature in ((np.int64(5), 2.0), (np.uint8(5), np.float32(2.0)), (torch.tensor(5), torch.tensor(2.0)), (5, np.float64(2.0)), (5, 2)):
        assert all(torch.equal(a, b) for a, b in zip(ops.top_logits(x, k, temperature=temperature), want))
    before = ops.launch_count()
    for k in (5.0, "5", None, np.float64(5)):
        with pytest.raises(ops.KernelError):
            ops.top_logits(x, k)
    assert ops.launch_count() == before
