"""Requests that ask something of their logits, and what goes wrong with them: submits refused, grammars shared or failing, biases that leave no
token. The engine stands above a step function that has no GPU."""

from __future__ import annotations


import numpy as np
import pytest

from research_2_b200.engine.scheduler import Full
from research_2_b200.sampling.controls import Controls
from tests.test_controls import controlled_engine
from tests.test_engine_protocol import VOCAB, continuation


class Turns:
    """Tokens of the residues 0, 1, 2 in turn."""

    def __init__(self, first: int = 0):
        self.n = first

    def allowed(self):
        return np.arange(VOCAB) % 3 == self.n % 3

    def advance(self, token):
        assert token % 3 == self.n % 3
        self.n += 1


class Wrong:
    """Answers with what it is given, or raises it; counts how often it is asked."""

    def __init__(self, answer):
        self.answer, self.asked = answer, 0

    def allowed(self):
        self.asked += 1
        if isinstance(self.answer, Exception):
            raise self.answer
        return self.answer

    def advance(self, token):
        pass


@pytest.mark.parametrize("answer,error", [(np.ones(VOCAB - 1, dtype=bool), ValueError), (np.zeros(3), ValueError), (OSError("no grammar"), OSError)])
def test_a_submit_that_is_refused_leaves_no_request_behind(answer, error):
    with controlled_engine(max_requests=1) as engine:
        with pytest.raises(error):
            engine.submit([5, 6], 4, controls=Controls(grammar=Wrong(answer)))
        assert not engine.has_work() and engine.request_events() == [] and not engine._controls.requests
        rid = engine.submit([5, 6], 4)
        assert engine.wait(rid).new_tokens == continuation([5, 6], 4)


def test_a_full_engine_does_not_ask_the_grammar():
    with controlled_engine(max_requests=1) as engine:
        first = engine.submit([5, 6], 2)
        grammar = Wrong(np.ones(VOCAB, dtype=bool))
        for _ in range(3):
            with pytest.raises(Full):
                engine.submit([7], 2, controls=Controls(grammar=grammar))
        assert grammar.asked == 0
        engine.wait(first)
        second = engine.submit([7], 2, controls=Controls(grammar=grammar))
        assert engine.wait(second).new_tokens == continuation([7], 2) and grammar.asked > 0
