"""Requests with controls and without in one engine: steps as graphs and launch by launch, alone and side by side, before and after. In float32 a
row's numbers do not depend on the batch or on how a step is launched, so tokens and log-probabilities are equal; in bfloat16 they may
round differently in another batch, so there the same batches are compared."""

from __future__ import annotations

import pytest

from tests.helpers import random_tokens
from tests.test_controls_gpu import asked_for, wide_a, wide_b  # noqa: F401

pytestmark = pytest.mark.gpu
PROMPTS = [(30, 0), (4, 1), (90, 2), (12, 3), (55, 4), (7, 5)]


def run_all(folder, vocab, which, temperature, **options):
    """Tokens and log-probabilities of the prompts in `which`, each with its own controls."""
    import research_2_b200 as r2

    prompts = [random_tokens(70 + i, PROMPTS[i][0], vocab) for i in which]
    records = {}
    with r2.run(folder, block_size=16, **options) as engine:
        rids = {}
        for i, prompt in zip(which, prompts):
            rids[i] = engine.submit(prompt, 10, temperature, top_k=0, seed=1000 + i, controls=asked_for(i, vocab))
        got = {i: engine.wait(rid).new_tokens for i, rid in rids.items()}
        for i, rid in rids.items():
            controls = asked_for(i, vocab)
            if controls is not None and controls.top_logprobs is not None:
                records[i] = engine.logprobs(rid)
    return got, records


@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_graphs_and_single_launches_give_the_same(wide_a, temperature):  # noqa: F811
    both = [run_all(wide_a, 512, range(6), temperature, dtype="float32", max_requests=6, capture=capture) for capture in (True, False)]
    assert both[0][0] == both[1][0]
    assert {i: [r.token for r in records] for i, records in both[0][1].items()} == {i: [r.token for r in records] for i, records in both[1][1].items()}
    assert both[0][1] == both[1][1]


@pytest.mark.parametrize("temperature", [0.0, 0.9])
@pytest.mark.parametrize("capture", [True, False])
def test_requests_side_by_side_get_what_they_get_alone(wide_a, temperature, capture):  # noqa: F811
    options = dict(dtype="float32", max_requests=6, capture=capture)
    together = run_all(wide_a, 512, range(6), temperature, **options)
    for i in range(6):
        alone = run_all(wide_a, 512, [i], temperature, **options)
        assert alone[0][i] == together[0][i], i
        assert alone[1].get(i) == together[1].get(i), i


@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_steps_without_controls_run_as_if_there_had_been_none(wide_b, temperature):  # noqa: F811
    """The same batches of bfloat16 rows in an engine that has never heard of controls, and in one whose controlled requests have ended: the same
    tokens, by the same launches of graphs."""
    import research_2_b200 as r2

    prompts = [random_tokens(90 + i, n, 1031) for i, n in enumerate((30, 4, 17))]

    def uncontrolled(engine):
        launched = []
        launch = engine.step_fn.launch_graph
        engine.step_fn.launch_graph = lambda batch: launched.append(launch(batch)) or launched[-1]
        rids = [engine.submit(p, 12, temperature, seed=i) for i, p in enumerate(prompts)]
        tokens = [engine.wait(rid).new_tokens for rid in rids]
        engine.step_fn.launch_graph = launch
        return tokens, [graph is not None for graph in launched]

    with r2.run(wide_b, dtype="bfloat16", max_requests=3) as engine:
        uncontrolled(engine)   # (graphs are made as shapes come)
        want = uncontrolled(engine)
        assert engine._controls is None
    with r2.run(wide_b, dtype="bfloat16", max_requests=3) as engine:
        uncontrolled(engine)
        rid = engine.submit(prompts[0], 5, temperature, seed=9, controls=asked_for(5, 1031))
        assert len(engine.wait(rid).new_tokens) == 5
        got = uncontrolled(engine)
        assert engine._controls is not None
    assert got == want and sum(want[1]) >= 10
