"""Requests that ask something of their logits, through the engine against the plain implementation; a teacher's lessons and a student that learns
from them."""

from __future__ import annotations

import json
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from tests.helpers import TINY_A, TINY_B, make_model_dir, random_tokens
from tests.plain import gpt2_plain
from tests.plain import logits_plain

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
DEV = "cuda:0"


def ops():
    from research_2_b200.kernels import ops as o

    return o


@pytest.fixture(scope="module")
def wide_a(tmp_path_factory):
    return make_model_dir(tmp_path_factory.mktemp("controls_a"), TINY_A, std=0.2)


@pytest.fixture(scope="module")
def wide_b(tmp_path_factory):
    return make_model_dir(tmp_path_factory.mktemp("controls_b"), TINY_B, std=0.2)


class EveryThird:
    """Tokens of one residue after another: what may come next depends on how many have come."""

    def __init__(self, vocab):
        self.vocab, self.n = vocab, 0

    def allowed(self):
        return np.arange(self.vocab) % 3 == self.n % 3

    def advance(self, token):
        assert token % 3 == self.n % 3
        self.n += 1


def asked_for(i: int, vocab: int):
    from research_2_b200.sampling.controls import Controls

    return [None, Controls(repetition_penalty=1.4, top_logprobs=3), Controls(presence_penalty=2.0, frequency_penalty=1.5),
            Controls(grammar=EveryThird(vocab), top_logprobs=0), Controls(logit_bias={7: 3.0, 9: -math.inf, 11: 1.5}, repetition_penalty=0.8),
            Controls(repetition_penalty=1.2, presence_penalty=0.5, logit_bias={3: 0.5}, grammar=EveryThird(vocab), top_logprobs=5)][i % 6]


def plain_continuation(folder, prompt, n, controls, vocab):
    """Greedy tokens and, beside each, the adjusted logits in 64 bits."""
    w, cfg = gpt2_plain.read_model(folder, torch.float32)
    grammar = EveryThird(vocab) if controls is not None and controls.grammar is not None else None
    answer, rows = [], []
    for _ in range(n):
        x = gpt2_plain.forward(w, cfg, torch.tensor(list(prompt) + answer))[-1].double().numpy()
        if controls is not None:
            x = logits_plain.adjust_row(x, prompt, answer, controls.repetition_penalty, controls.presence_penalty, controls.frequency_penalty,
                                        sorted((controls.logit_bias or {}).items()), grammar.allowed() if grammar else None)
        token = int(np.argmax(x))
        if grammar:
            grammar.advance(token)
        answer.append(token)
        rows.append(x)
    return answer, rows


@pytest.mark.parametrize("options", [dict(max_requests=6), dict(max_requests=3, max_batch_tokens=32), dict(max_requests=6, num_slabs=14, block_size=16),
                                     dict(max_requests=4, capture=True)])
def test_generation_with_controls_against_the_plain_implementation(wide_a, options):
    import research_2_b200 as r2
    from research_2_b200.engine.api import generate_with

    vocab, n = 512, 14
    prompts = [random_tokens(40 + i, length, vocab) for i, length in enumerate((5, 33, 1, 17, 60, 9))]
    want = [plain_continuation(wide_a, p, n, asked_for(i, vocab), vocab) for i, p in enumerate(prompts)]
    records = {}
    with r2.run(wide_a, dtype="float32", block_size=options.pop("block_size", 16), **options) as engine:
        got = generate_with(engine, prompts, n, stop_token_ids=(), controls=[asked_for(i, vocab) for i in range(6)],
                            ended=lambda i, rid: records.update({i: engine.logprobs(rid)}) if i else None)
    for i in range(6):
        answer = want[i][0]
        stop = answer.index(511) + 1 if 511 in answer else n   # (the model's own end token)
        assert got[i] == answer[:stop], i
    for i in (1, 3, 5):
        n_top = asked_for(i, vocab).top_logprobs
        assert [r.token for r in records[i]] == got[i]
        for record, x in zip(records[i], want[i][1]):
            log_p = x - (x.max() + math.log(np.exp(x - x.max()).sum()))
            # logits of size 10 to 20 in float32 through two layers: 1e-4
            assert abs(record.logprob - log_p[record.token]) < 1e-3 and len(record.top) == n_top
            for token, value in record.top:
                if math.isfinite(value):
                    assert abs(value - log_p[token]) < 1e-3
            assert list(record.top) == sorted(record.top, key=lambda t: -t[1])


def test_controls_run_beside_graphs_in_bfloat16(wide_b):
    """Steps as graphs and launch by launch give the same tokens; requests without controls get what they get alone."""
    import research_2_b200 as r2

    vocab = 1031
    prompts = [random_tokens(70 + i, length, vocab) for i, length in enumerate((30, 4, 90, 12, 55, 7))]
    runs = [r2.generate(wide_b, prompts, 10, dtype="bfloat16", max_requests=6, capture=capture, temperature=0.7, seed=3,
                        controls=[asked_for(i, vocab) for i in range(6)]) for capture in (True, False)]
    assert [t % 3 for t in runs[0][3]] == [i % 3 for i in range(10)]
    assert 9 not in runs[0][4]
    # graphs and single launches of bfloat16 products may round differently; what the controls rule holds in both
    assert [t % 3 for t in runs[1][5]] == [i % 3 for i in range(10)]
    with r2.run(wide_b, dtype="bfloat16", max_requests=2) as engine:
        free = engine.submit(prompts[0], 8)
        alone = engine.wait(free).new_tokens
        a, b = engine.submit(prompts[0], 8), engine.submit(prompts[1], 8, controls=asked_for(1, vocab))
        together = engine.wait(a).new_tokens
        engine.wait(b)
        assert len(engine.logprobs(b)) == 8
    assert len(together) == len(alone) == 8


def test_sampling_draws_from_what_is_allowed(wide_a):
    import research_2_b200 as r2
    from research_2_b200.sampling.controls import AllowedTokens, Controls

    allowed = [3, 100, 257, 509]
    got = r2.generate(wide_a, [[5, 6, 7]] * 4, 12, temperature=1.5, seed=1, dtype="float32", controls=Controls(grammar=AllowedTokens(allowed, 512)))
    assert {t for g in got for t in g} <= set(allowed) and len({tuple(g) for g in got}) > 1
    only = r2.generate(wide_a, [[5, 6, 7]], 5, top_k=40, temperature=1.0, dtype="float32", controls=Controls(grammar=AllowedTokens([77], 512)))
    assert only == [[77] * 5]


def test_keep_tokens():
    history = torch.full((4, 10), -1, dtype=torch.int32, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ops().keep_tokens(history, i32([5, 6, 7, 8, 9, 10]), i32([0, 1, 9, 10, 2, 3]), i32([0, 0, 1, 1, -1, 2]), i32([2, 0, 9]))
    want = torch.full((4, 10), -1, dtype=torch.int32)
    want[2, 0], want[2, 1], want[0, 9] = 5, 6, 7   # a place beyond the table, a pad row and a slot beyond it are left out
    assert torch.equal(history.cpu(), want)
    with pytest.raises(ops().KernelError):
        ops().keep_tokens(history, i32([1, 2]), i32([0]), i32([0, 0]), i32([0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,offset", [(1, 0), (7, 3), (2049, 1), (50257, 0)])
def test_scale_rows(dtype, vocab, offset):
    buf = torch.randn(5, vocab + offset + 2, device=DEV).to(dtype)
    x, before = buf[:, offset: offset + vocab], buf.clone()
    factors = torch.tensor([1.0, 0.5, -3.0, 0.0, 1.7], device=DEV)
    got = ops().scale_rows(x, factors)
    want = (before[:, offset: offset + vocab].float() * factors[:, None]).to(dtype)
    assert got.data_ptr() == x.data_ptr() and torch.equal(x, want)
    assert torch.equal(buf[:, :offset], before[:, :offset]) and torch.equal(buf[:, offset + vocab:], before[:, offset + vocab:])
    ops().scale_rows(x, torch.tensor(2.0, device=DEV))
    assert torch.equal(x, (want.float() * 2).to(dtype))


@pytest.mark.parametrize("portion", [1024, 7])
def test_teach_is_the_top_of_what_replay_writes(wide_b, portion):
    import research_2_b200 as r2
    from research_2_b200.engine.replay import Replay

    sequences = [random_tokens(i, n, 1031) for i, n in enumerate((40, 1, 23))]
    lessons = r2.teach(wide_b, sequences, 12, 2.0, dtype="float32", portion=portion)
    replay = Replay(str(wide_b), "float32", 64, max_live=1)
    for tokens, lesson in zip(sequences, lessons):
        logits = replay.step({"entries": [{"id": 0, "tokens": tokens, "want": list(range(len(tokens)))}], "end": [0]})
        assert lesson.ids.shape == (len(tokens), 12) and lesson.tokens.tolist() == tokens
        for t in range(len(tokens)):
            values, ids, log_sum = logits_plain.top_row(logits[t], 12, 2.0)
            assert lesson.ids[t].tolist() == ids and np.array_equal(lesson.teacher[t].astype(np.float64), values)
            assert abs(lesson.log_sum[t] - log_sum) < 1e-5
    with pytest.raises(ValueError):
        r2.teach(wide_b, [[]], 12)


def plain_loss(logits, ids, teacher, log_sum, temperature, weight):
    """The loss in torch's own operations, for its gradients."""
    log_q = torch.log_softmax(logits / temperature, dim=1)
    p = torch.exp(teacher / temperature - log_sum[:, None])
    listed = torch.gather(log_q, 1, ids.long())
    others = torch.ones_like(log_q).scatter(1, ids.long(), 0.0)
    rest_q, rest_p = (torch.exp(log_q) * others).sum(1), (1 - p.sum(1)).clamp(min=0)
    kl = (p * (torch.log(p) - listed)).sum(1) + torch.where(rest_p > 0, rest_p * (torch.log(rest_p) - torch.log(rest_q)), 0.0)
    return weight * temperature**2 * kl


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_loss_with_torch_gradients(dtype):
    import research_2_b200 as r2

    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(9, 1031, generator=gen) * 3).to(dtype).to(DEV)
    values, ids, log_sum = ops().top_logits((torch.randn(9, 1031, generator=gen) * 3).to(DEV), 20, temperature=1.5)
    weight = torch.rand(9, generator=gen).to(DEV) + 0.5
    above = torch.tensor([1.0, 2.0, 0.0, 1.0, -1.0, 1.0, 0.5, 1.0, 3.0], device=DEV)
    leaf = x.clone().requires_grad_()
    loss = r2.distill_loss(leaf, ids, values, log_sum=log_sum, temperature=1.5, weight=weight)
    (loss * above).sum().backward()
    other = x.double().requires_grad_()
    want = plain_loss(other, ids, values.double(), log_sum.double(), 1.5, weight.double())
    (want * above.double()).sum().backward()
    assert torch.allclose(loss.double(), want, rtol=1e-5, atol=1e-5)
    # a gradient's numbers are below weight * temperature * 3 = 7; in bfloat16 they are rounded, and once more where a factor scales them
    assert leaf.grad.dtype == dtype
    assert torch.all((leaf.grad.double() - other.grad).abs() <= 7e-5 + (2.0**-7 * other.grad.abs() if dtype == torch.bfloat16 else 0))
    with torch.no_grad():
        assert torch.equal(r2.distill_loss(leaf, ids, values, log_sum=log_sum, temperature=1.5, weight=weight) > 0, loss > 0)


def test_a_student_learns_from_a_teacher(wide_b):
    """The whole way: a model of the engine teaches, a table of next-token logits per token (a student of two matrices) learns from its top
    logits, and drafts more of the teacher's own answers than it did."""
    import research_2_b200 as r2

    vocab, tau = 1031, 1.0
    prompts = [random_tokens(i, 8, vocab) for i in range(24)]
    answers = r2.generate(wide_b, prompts, 40, temperature=1.0, seed=5, dtype="bfloat16", max_requests=24)
    sequences = [p + a for p, a in zip(prompts, answers)]
    lessons = r2.teach(wide_b, sequences, 32, tau, dtype="bfloat16")
    tokens = torch.tensor(np.concatenate([le.tokens for le in lessons]), device=DEV).long()
    ids, teacher, log_sum = (torch.tensor(np.concatenate([getattr(le, name) for le in lessons]), device=DEV) for name in ("ids", "teacher", "log_sum"))
    torch.manual_seed(0)
    table = torch.nn.Embedding(vocab, 64, device=DEV)
    head = torch.nn.Linear(64, vocab, device=DEV)
    optimizer = torch.optim.Adam([*table.parameters(), *head.parameters()], lr=2e-2)
    weight = torch.full((len(tokens),), 1.0 / len(tokens), device=DEV)
    losses = []
    for _ in range(40):
        logits = head(table(tokens))
        loss = r2.distill_loss(logits, ids, teacher, log_sum=log_sum, temperature=tau, weight=weight).sum()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.6 * losses[0], losses
    drafted = head(table(tokens)).argmax(dim=1)
    assert float((drafted == ids[:, 0]).float().mean()) > 0.2


def test_command_line_controls_and_lessons(wide_a, tmp_path):
    def run(*args):
        out = subprocess.run([sys.executable, "-m", "research_2_b200", *args], cwd=ROOT, capture_output=True, text=True, timeout=600)
        assert out.returncode == 0, out.stderr
        return out.stdout

    lines = run("generate", "--model", str(wide_a), "--prompt-tokens", "5,17,3", "--max-new-tokens", "6", "--dtype", "float32", "--allow-tokens", "7,8,9",
                "--presence-penalty", "50", "--logit-bias", "8:-inf")
    tokens = json.loads(lines.splitlines()[-1])["tokens"]
    assert set(tokens) <= {7, 9} and set(tokens[:2]) == {7, 9}
    path = tmp_path / "lesson.npz"
    run("teach", "--model", str(wide_a), "--tokens", "5,17,3", "--tokens", "9", "--top", "4", "--temperature", "2", "--dtype", "float32", "--out", str(path))
    with np.load(path) as lesson:
        assert lesson["ids_0"].shape == (3, 4) and lesson["teacher_1"].shape == (1, 4) and float(lesson["temperature"]) == 2.0
        assert lesson["tokens_0"].tolist() == [5, 17, 3]
