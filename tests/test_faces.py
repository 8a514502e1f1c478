"""Operators called with tensors in one step (`csrc/faces`): without a GPU, what they leave to the caller's checks."""

from __future__ import annotations

import pytest
import torch

from research_2_b200.csrc.build import faces_module


def test_faces_leave_what_is_not_plain():
    faces, x = faces_module(), torch.zeros(2, 40)
    assert faces.top_logits(x, 3, 1.0, 0) is None
    assert faces.top_logits(None, 3, 1.0, 0) is None
    assert faces.top_logits() is None and faces.adjust_logits(x) is None and faces.distill(x) is None
    assert faces.adjust_logits(x, *[None] * 13) is None
    assert faces.distill(x, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3), None, 1.0, None, True, None, 0) is None


def test_faces_are_bound_by_name():
    faces = faces_module()
    with pytest.raises(ValueError):
        faces.bind("no such operator", 8)
    with pytest.raises(TypeError):
        faces.bind("top_logits")
