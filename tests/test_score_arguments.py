"""Sequences that scoring and teaching refuse before they load a model."""

import numpy as np
import pytest
import torch

import research_2_b200 as r2


@pytest.mark.parametrize("sequence", [np.array([3, 2**32 + 5]), np.array([-(2**32) + 1, 7]), torch.tensor([2**31, 1]), [1, 2**40], [1, 2**70], [1.5, 2.0], np.array([3.0, 4.0]), ["1", "2"]])
def test_tokens_that_32_bits_would_make_others_of(sequence, tmp_path):
    """A cut to 32 bits, or to a whole number, names another token, whose score would be the answer."""
    for call in (lambda: r2.score(tmp_path / "no model", [[1, 2], sequence]), lambda: r2.teach(tmp_path / "no model", [[1, 2], sequence])):
        with pytest.raises(ValueError, match="sequence 1"):
            call()
