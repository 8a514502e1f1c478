"""What requests ask of their logits, on the host: the checks, the masks' words, what a step's rows are packed into, and the engine above a step
function that has no GPU and applies the packed numbers by their definition."""

from __future__ import annotations

import math

import numpy as np
import pytest

from research_2_b200.engine.controls import StepControls, _Request, allowed_words, pack_rows
from research_2_b200.sampling.controls import AllowedTokens, Controls, NoTokenAllowed, TokenLogprobs, mask_words, pack_mask
from tests.test_engine_protocol import VOCAB, make_engine


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 211, 1031])
def test_pack_mask_puts_token_t_at_bit_t(vocab):
    rng = np.random.default_rng(vocab)
    allowed = rng.random(vocab) < 0.5
    words = pack_mask(allowed)
    assert words.dtype == np.int32 and words.shape == (mask_words(vocab),)
    bits = [(int(words.view(np.uint32)[t // 32]) >> (t % 32)) & 1 for t in range(vocab)]
    assert bits == allowed.astype(int).tolist()
    grammar = AllowedTokens(np.flatnonzero(allowed) if allowed.any() else [0], vocab)
    assert np.array_equal(allowed_words(grammar, vocab), words if allowed.any() else pack_mask(np.arange(vocab) == 0))


def test_allowed_words_of_truth_values_and_of_words():
    class Grammar:
        def __init__(self, value):
            self.value = value

        def allowed(self):
            return self.value

    allowed = np.arange(40) % 3 == 0
    assert np.array_equal(allowed_words(Grammar(allowed), 40), pack_mask(allowed))
    words = pack_mask(allowed)
    words[-1] |= np.int32(1 << 20)   # beyond the vocabulary
    assert np.array_equal(allowed_words(Grammar(words.view(np.uint32)), 40), pack_mask(allowed))
    for bad in (allowed[:-1], words[:-1], words.astype(np.int64), np.zeros(40, dtype=np.float32)):
        with pytest.raises(ValueError):
            allowed_words(Grammar(bad), 40)


@pytest.mark.parametrize("bad", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.nan),
                                 dict(presence_penalty=math.inf), dict(frequency_penalty=math.nan), dict(logit_bias={100: 1.0}), dict(logit_bias={-1: 1.0}),
                                 dict(logit_bias={1.5: 1.0}), dict(logit_bias={1: math.nan}), dict(logit_bias={1: math.inf}), dict(grammar=object()),
                                 dict(top_logprobs=-1), dict(top_logprobs=101)])
def test_controls_refuse(bad):
    with pytest.raises(ValueError):
        Controls(**bad).checked(100)


def test_controls_know_whether_anything_is_asked_for():
    assert not Controls() and not Controls(logit_bias={})
    for asked in (dict(repetition_penalty=1.1), dict(presence_penalty=-0.5), dict(frequency_penalty=0.1), dict(logit_bias={3: -math.inf}),
                  dict(grammar=AllowedTokens([1], 9)), dict(top_logprobs=0)):
        assert Controls(**asked).checked(9)


def request(vocab, n_prompt=3, mask=None, **asked) -> _Request:
    controls = Controls(**asked)
    biases = sorted((controls.logit_bias or {}).items())
    return _Request(controls, n_prompt, np.array([t for t, _ in biases], dtype=np.int32), np.array([v for _, v in biases], dtype=np.float32), mask)


def test_pack_rows_is_neutral_where_nothing_is_asked():
    vocab = 70
    mask = pack_mask(np.arange(vocab) % 2 == 0)
    rows = [None, request(vocab, 5, repetition_penalty=1.5, logit_bias={7: 2.0, 3: -math.inf}), request(vocab, mask=mask, presence_penalty=0.25), None,
            request(vocab, frequency_penalty=0.5, logit_bias={69: 1.0})]
    packed, parts = pack_rows(rows, vocab)

    def part(name):
        first, count, kind = parts[name]
        assert first % 4 == 0
        return packed[first: first + count].view(kind).tolist()

    assert part("prompt_lengths") == [0, 5, 3, 0, 3] and part("repetition") == [1.0, 1.5, 1.0, 1.0, 1.0]
    assert part("presence") == [0.0, 0.0, 0.25, 0.0, 0.0] and part("frequency") == [0.0, 0.0, 0.0, 0.0, 0.5]
    assert part("mask_rows") == [-1, -1, 0, -1, -1] and part("mask") == mask.tolist()
    assert part("bias_start") == [0, 0, 2, 2, 2, 3] and part("bias_ids") == [3, 7, 69] and part("bias_values") == [-math.inf, 2.0, 1.0]


class HostControls(StepControls):
    """The same book-keeping; the pass is the fake step function's: its token is the likeliest, shifted where the grammar forbids it."""

    def step(self, batch, plan):
        graph = self.step_fn.launch_graph(batch)
        tokens = graph.tokens_on_host(plan.n_entries).copy()
        self._top = [np.zeros((plan.n_entries, 2), np.float32), np.zeros((plan.n_entries, 2), np.int32), np.ones(plan.n_entries, np.float32),
                     np.zeros(plan.n_entries, np.float32)]
        self.seen = getattr(self, "seen", []) + [[int(r) for r in plan.req]]
        for e, (rid, emits) in enumerate(zip(plan.req, plan.emits)):
            r = self.requests.get(int(rid))
            if r is None or not emits or r.mask is None:
                continue
            while not (int(r.mask.view(np.uint32)[tokens[e] // 32]) >> (int(tokens[e]) % 32)) & 1:
                tokens[e] = (tokens[e] + 1) % VOCAB
        return tokens


def controlled_engine(**options):
    engine = make_engine(**options)
    engine._controls = HostControls(engine.step_fn, 3, 96, VOCAB)
    return engine


def test_engine_holds_a_request_to_its_grammar_and_leaves_the_others_alone():
    from research_2_b200.engine.api import generate_with
    from tests.test_engine_protocol import PROMPTS, continuation

    class Rising:
        """Each token is larger than the one before; the last allows nothing more."""

        def __init__(self):
            self.last, self.told = 0, []

        def allowed(self):
            return np.arange(VOCAB) > self.last

        def advance(self, token):
            self.told.append(token)
            self.last = token

    grammar = Rising()
    with controlled_engine() as engine:
        ended = []
        got = generate_with(engine, PROMPTS, 6, controls=[Controls(grammar=grammar, top_logprobs=1) if i == 0 else None for i in range(len(PROMPTS))],
                            ended=lambda i, rid: ended.append((i, engine.logprobs(rid) if i == 0 else None)))
        assert not engine._controls.requests
    assert got[1:] == [continuation(p, 6) for p in PROMPTS[1:]]
    assert got[0] == sorted(set(got[0])) == grammar.told and len(got[0]) == 6
    records = dict(ended)[0]
    assert [r.token for r in records] == got[0] and records[0] == TokenLogprobs(got[0][0], -1.0, ((0, -1.0),))
    assert sorted(i for i, _ in ended) == list(range(len(PROMPTS)))


def test_a_grammar_that_allows_nothing_is_said_before_the_next_plan():
    class Once:
        def __init__(self):
            self.left = True

        def allowed(self):
            return np.full(VOCAB, self.left)

        def advance(self, token):
            self.left = False

    with controlled_engine() as engine:
        rid = engine.submit([5, 6, 7], max_new_tokens=4, controls=Controls(grammar=Once()))
        other = engine.submit([9], max_new_tokens=3)
        engine.step()
        with pytest.raises(NoTokenAllowed) as raised:
            engine.step()
        assert raised.value.req_id == rid
        engine.cancel(rid)
        assert len(engine.wait(other).new_tokens) == 3
        with pytest.raises(KeyError):
            engine.logprobs(rid)


def test_ids_that_are_given_again_start_without_controls():
    with controlled_engine(max_requests=1) as engine:
        a = engine.submit([5, 6], max_new_tokens=2, controls=Controls(top_logprobs=1))
        engine.wait(a)
        assert len(engine.logprobs(a)) == 2
        b = engine.submit([5, 6], max_new_tokens=2)
        assert b == a
        with pytest.raises(KeyError):
            engine.logprobs(b)
        n = len(engine._controls.seen)
        engine.wait(b)
        assert len(engine._controls.seen) == n, "a step without controlled requests runs as it always does"
        with pytest.raises(ValueError):
            engine.submit([1], max_new_tokens=1, controls=Controls(repetition_penalty=0.0))
        assert not engine.has_work()


def test_generate_refuses_controls_of_another_number():
    from research_2_b200.engine.api import generate_with

    with controlled_engine() as engine, pytest.raises(ValueError):
        generate_with(engine, [[1], [2]], 2, controls=[Controls()])
