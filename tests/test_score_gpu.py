"""Scores of given tokens through the engine: against the head's own hidden rows in 64 bits, against the logits that a replay writes, in portions, with capped
logits, through the command line."""

from __future__ import annotations

import json
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.helpers import TINY_B, TINY_C, make_model_dir, random_tokens
from tests.plain.vocabulary_plain import Loss

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def wide_b(tmp_path_factory):
    return make_model_dir(tmp_path_factory.mktemp("score_b"), TINY_B, std=0.2)


@pytest.fixture(scope="module")
def wide_c(tmp_path_factory):
    return make_model_dir(tmp_path_factory.mktemp("score_c"), TINY_C, std=0.2)


@pytest.mark.parametrize("portion", [2048, 16])
def test_scores_are_those_of_the_logits(wide_b, portion):
    import research_2_b200 as r2
    from research_2_b200.engine.replay import Replay

    sequences = [random_tokens(i, n, 1031) for i, n in enumerate((40, 1, 2, 33))]
    scores = r2.score(wide_b, sequences, dtype="float32", portion=portion)
    replay = Replay(str(wide_b), "float32", 64, max_live=1)
    for tokens, got in zip(sequences, scores):
        assert got.dtype == np.float32 and got.shape == (len(tokens) - 1,)
        if len(tokens) == 1:
            continue
        logits = replay.step({"entries": [{"id": 0, "tokens": tokens, "want": list(range(len(tokens)))}], "end": [0]}).astype(np.float64)
        log_q = logits - np.logaddexp.reduce(logits, axis=1, keepdims=True)
        want = np.array([log_q[t, tokens[t + 1]] for t in range(len(tokens) - 1)])
        # two sums of 96 products each on both sides (below 96 * 3 * 1 in size): (4 * 96 + 16) units of 2^-24 of it, twice, and 1e-5 for the exponentials
        assert np.abs(got - want).max() <= 2 * (4 * 96 + 16) * 2.0**-24 * 288 + 1e-5


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_are_those_of_the_heads_rows(wide_c, dtype, monkeypatch):
    import research_2_b200 as r2
    from research_2_b200.kernels import ops

    seen, real = [], ops.token_loss

    def kept(hidden, table, targets, **kwargs):
        out = real(hidden, table, targets, **kwargs)
        seen.append((hidden.clone(), table, targets.clone(), out[0].clone(), kwargs))
        return out

    monkeypatch.setattr(ops, "token_loss", kept)
    sequences = [random_tokens(i + 5, n, 777) for i, n in enumerate((300, 150))]
    scores = r2.score(wide_c, sequences, dtype=dtype, portion=130)
    assert [len(s) for s in seen and scores] == [299, 149]
    rows = 0
    for hidden, table, targets, loss, kwargs in seen:
        assert hidden.dtype == getattr(torch, dtype) and hidden.shape[0] <= 130
        want = Loss(hidden, table, targets, softcap=kwargs.get("softcap", 0.0))
        assert torch.all((loss.double() - want.loss).abs() <= want.loss_off)
        rows += hidden.shape[0]
    assert rows == 299 + 149
    assert np.array_equal(np.concatenate(scores), -torch.cat([s[3] for s in seen]).cpu().numpy())
    assert [t for s in seen for t in s[2].tolist()] == sequences[0][1:] + sequences[1][1:]


def test_scores_of_a_model_with_capped_logits(tmp_path):
    import research_2_b200 as r2
    from research_2_b200.engine.replay import Replay
    from tests import lagelorn_cases

    case = next(c for c in lagelorn_cases.CASES.values() if c["config"].get("logit_softcap"))
    folder = lagelorn_cases.make_model_dir(tmp_path / "capped", case)
    replay = Replay(str(folder), "float32", 64, max_live=1)
    vocab, cap = replay.model.vocab_size, replay.model.spec.logit_softcap
    assert cap > 0
    tokens = random_tokens(3, 30, vocab)
    (got,) = r2.score(folder, [tokens], dtype="float32")
    logits = replay.step({"entries": [{"id": 0, "tokens": tokens, "want": list(range(30))}], "end": [0]}).astype(np.float64)
    log_q = logits - np.logaddexp.reduce(logits, axis=1, keepdims=True)
    # logits below the cap; float32 sums of at most a few hundred products, and the two tanh's errors of 16 units of the cap
    assert np.abs(got - log_q[np.arange(29), tokens[1:]]).max() <= 1e-4 + 64 * 2.0**-24 * cap


def test_what_cannot_be_scored(wide_b):
    import research_2_b200 as r2

    for bad in ([[]], [[1, 1031]], [[-1, 2]]):
        with pytest.raises(ValueError):
            r2.score(wide_b, bad)
    with pytest.raises(ValueError):
        r2.score(wide_b, [[1, 2]], portion=0)
    assert r2.score(wide_b, []) == [] and [len(s) for s in r2.score(wide_b, [[4]])] == [0]


def test_command_line(wide_b):
    import research_2_b200 as r2

    out = subprocess.run([sys.executable, "-m", "research_2_b200", "score", "--model", str(wide_b), "--tokens", "5,17,3", "--tokens", "9", "--dtype", "float32"],
                         cwd=ROOT, capture_output=True, text=True, check=True).stdout
    lines = [json.loads(line) for line in out.splitlines()]
    assert [line["tokens"] for line in lines] == [[5, 17, 3], [9]]
    want = r2.score(wide_b, [[5, 17, 3]], dtype="float32")[0]
    assert lines[0]["log_probs"] == [float(p) for p in want] and lines[1]["log_probs"] == []
