"""float32 scores are the same bits however a sequence is cut, as float32 logits are: losses of few rows have a kernel of their own, which these scores do not go through."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.helpers import TINY_B, make_model_dir, random_tokens
from tests.test_token_loss_gpu import BF16, DEV, F32, Case, ops

pytestmark = pytest.mark.gpu


def test_float32_scores_do_not_depend_on_the_portion(tmp_path):
    import research_2_b200 as r2

    model = make_model_dir(tmp_path, TINY_B, std=0.2)
    tokens = random_tokens(3, 201, 1031)
    whole = r2.score(model, [tokens], dtype="float32")[0]
    for portion in (1, 7, 64, 128, 129, 150):
        assert np.array_equal(r2.score(model, [tokens], dtype="float32", portion=portion)[0], whole)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width,vocab,softcap", [(96, 1031, 0.0), (100, 5000, 20.0), (1000, 700, 0.0)])
def test_rows_alike(dtype, width, vocab, softcap):
    c = Case(300, width, vocab, dtype, 3, softcap=softcap)
    whole = ops().token_loss(c.hidden, c.table, c.targets, weight=c.weight, softcap=softcap)
    for first, last in ((0, 300), (0, 1), (10, 138), (10, 139), (172, 300), (290, 300)):
        part = ops().token_loss(c.hidden[first: last], c.table, c.targets[first: last], weight=c.weight[first: last], softcap=softcap, alike=True)
        assert all(torch.equal(a, b[first: last]) for a, b in zip(part, whole))
