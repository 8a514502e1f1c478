"""Requests that ask something of their logits, and what goes wrong with them: submits refused, grammars shared or failing, biases that leave no
token. The engine stands above a step function that has no GPU."""

from __future__ import annotations

import math

import numpy as np
import pytest

from research_2_b200.engine.api import generate_with
from research_2_b200.engine.scheduler import Full
from research_2_b200.sampling.controls import AllowedTokens, Controls, NoTokenAllowed
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


@pytest.mark.parametrize("max_requests", [1, 2, 3])
@pytest.mark.parametrize("as_list", [False, True])
def test_a_grammar_for_several_prompts_follows_each_of_them(max_requests, as_list):
    prompts = [[5, 6], [7], [8, 9, 10], [11]]
    controls = Controls(grammar=Turns(1), top_logprobs=1)
    with controlled_engine(max_requests=max_requests) as engine:
        got = generate_with(engine, prompts, 6, controls=[controls, None, controls, controls] if as_list else controls)
    assert controls.grammar.n == 1, "the one that was given is told nothing"
    for i, tokens in enumerate(got):
        if as_list and i == 1:
            assert tokens == continuation(prompts[1], 6)
        else:
            assert [t % 3 for t in tokens] == [1, 2, 0, 1, 2, 0]


def test_a_prompt_s_own_grammar_is_told_what_came():
    own, other = Turns(), Turns(2)
    with controlled_engine() as engine:
        got = generate_with(engine, [[5], [6]], 4, controls=[Controls(grammar=own), Controls(grammar=other)])
    assert (own.n, other.n) == (4, 6) and [t % 3 for t in got[1]] == [2, 0, 1, 2]


def test_a_grammar_that_follows_a_request_is_refused_for_another():
    shared = Turns()
    allowed = AllowedTokens([3, 4, 5], VOCAB)
    with controlled_engine(max_requests=4) as engine:
        a = engine.submit([5], 3, controls=Controls(grammar=shared))
        with pytest.raises(ValueError, match="another request"):
            engine.submit([6], 3, controls=Controls(grammar=shared))
        b, c = (engine.submit([6], 2, controls=Controls(grammar=allowed)) for _ in range(2))
        assert len(engine.wait(a).new_tokens) == 3 and len(engine.wait(b).new_tokens) == len(engine.wait(c).new_tokens) == 2
        again = engine.submit([6], 3, controls=Controls(grammar=shared))   # (its request has ended)
        assert [t % 3 for t in engine.wait(again).new_tokens] == [0, 1, 2]
        assert not engine.has_work()


@pytest.mark.parametrize("controls", [dict(grammar=AllowedTokens([7, 9], VOCAB), logit_bias={7: -math.inf, 9: -math.inf, 3: 1.0}),
                                      dict(logit_bias=dict.fromkeys(range(VOCAB), -math.inf))])
def test_biases_that_leave_no_token_are_said_before_the_next_plan(controls):
    with controlled_engine() as engine:
        rid = engine.submit([5, 6], 4, controls=Controls(**controls, top_logprobs=1))
        other = engine.submit([9], 3)
        for _ in range(2):
            with pytest.raises(NoTokenAllowed) as raised:
                engine.step()
            assert raised.value.req_id == rid
        engine.cancel(rid)
        assert engine.wait(other).new_tokens == continuation([9], 3)


def test_biases_that_leave_a_token_are_no_error():
    some = {t: -math.inf for t in range(VOCAB) if t != 40}
    with controlled_engine() as engine:
        a = engine.submit([5, 6], 3, controls=Controls(logit_bias=some))
        b = engine.submit([5, 6], 3, controls=Controls(grammar=AllowedTokens([40, 41], VOCAB), logit_bias={41: -math.inf, 40: -5.0}))
        assert len(engine.wait(a).new_tokens) == len(engine.wait(b).new_tokens) == 3


def test_a_grammar_that_comes_to_what_biases_forbid():
    class Narrowing(Turns):
        def allowed(self):
            return np.arange(VOCAB) == 50 + self.n

        def advance(self, token):
            self.n += 1

    with controlled_engine() as engine:
        rid = engine.submit([5, 6], 9, controls=Controls(grammar=Narrowing(), logit_bias={52: -math.inf}))
        engine.step()
        engine.step()
        with pytest.raises(NoTokenAllowed):
            engine.step()
        assert engine.poll(rid).new_tokens == [50, 51]
        engine.cancel(rid)


@pytest.mark.parametrize("when", ["told", "asked"])
def test_a_grammar_that_fails_fails_alone(when):
    """What one request's grammar raises is raised by the step, and again until the request is cancelled; the others' grammars and records go on."""
    class Failing(Turns):
        def advance(self, token):
            super().advance(token)
            if when == "told" and self.n == 2:
                raise OSError("lost")

        def allowed(self):
            if when == "asked" and self.n == 2:
                raise OSError("lost")
            return super().allowed()

    other = Turns(1)
    with controlled_engine() as engine:
        engine.keep_events = True
        bad = engine.submit([5, 6], 6, controls=Controls(grammar=Failing()))
        good = engine.submit([7], 6, controls=Controls(grammar=other, top_logprobs=1))
        engine.step()
        for _ in range(3):
            with pytest.raises(OSError, match="lost"):
                engine.step()
        assert other.n == 3 and len(engine.logprobs(good)) == 2 and len(engine.events) == 2
        assert [t % 3 for t in engine.poll(bad).new_tokens] == [0, 1]
        engine.cancel(bad)
        assert [t % 3 for t in engine.wait(good).new_tokens] == [1, 2, 0, 1, 2, 0]
        assert [r.token % 3 for r in engine.logprobs(good)] == [1, 2, 0, 1, 2, 0]


def test_a_grammar_that_fails_at_its_last_token():
    class Failing(Turns):
        def advance(self, token):
            super().advance(token)
            if self.n == 2:
                raise OSError("lost")

    with controlled_engine() as engine:
        bad, other = engine.submit([5, 6], 2, controls=Controls(grammar=Failing())), engine.submit([9], 4)
        engine.step()
        with pytest.raises(OSError):
            engine.step()
        assert engine.poll(bad).finished and engine.wait(other).new_tokens == continuation([9], 4)


def test_plans_by_hand_refuse_requests_with_controls():
    with controlled_engine() as engine:
        rid = engine.submit([5, 6], 2, controls=Controls(grammar=Turns()))
        with pytest.raises(RuntimeError, match="only step"):
            engine.plan()
        engine.step()
        engine.step()
        other = engine.submit([9], 2)
        plan = engine.plan()   # (the one with controls has ended, polled or not)
        assert plan.n_entries == 1 and engine.build_batch(plan).n_entries == 1
        engine.commit([3])
        assert engine.poll(rid).finished and engine.wait(other).new_tokens[0] == 3
