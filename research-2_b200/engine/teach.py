"""A model as a teacher: given sequences of tokens, each position's largest next-token logits, for a student to learn from
(`sampling.distill.distill_loss`) or to compare itself with. Sequences pass through the engine's step function in portions, as prompts do,
and a row's logits are reduced on the device: 64 of 50,257 logits a row are 512 bytes where all of them are 200 KB."""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from .replay import Replay, token_sequences


@dataclass(frozen=True)
class Lesson:
    """Row t belongs to what follows tokens[: t + 1]: `teacher` float32 [T, K] the largest logits, `ids` int32 [T, K] their tokens, `log_sum` float32 [T]
    the logarithm of the sum of exp(logits / temperature)."""

    tokens: np.ndarray
    ids: np.ndarray
    teacher: np.ndarray
    log_sum: np.ndarray
    temperature: float


def teach(model_dir, sequences, k: int = 64, temperature: float = 1.0, *, dtype: str = "bfloat16", device: str = "cuda:0", portion: int = 1024,
          block_size: int = 16) -> list[Lesson]:
    """A lesson for each sequence of token ids. `portion`: rows of a step (their logits are on the device at a time)."""
    sequences = token_sequences(sequences)
    if portion < 1:
        raise ValueError(f"portion must be >= 1, got {portion}")
    if not sequences:
        return []
    replay = Replay(str(model_dir), dtype, max(len(s) for s in sequences), block_size, device, max_live=1)
    lessons = []
    for n, tokens in enumerate(sequences):
        parts = []
        for begin in range(0, len(tokens), portion):
            rows = tokens[begin: begin + portion]
            entry = {"id": n, "tokens": rows.tolist(), "want": list(range(len(rows)))}
            parts.append(replay.step_top({"entries": [entry], "end": [n] if begin + portion >= len(tokens) else []}, k, temperature))
        teacher, ids, log_sum = (np.concatenate(column) for column in zip(*parts))
        lessons.append(Lesson(tokens, ids, teacher, log_sum, temperature))
    return lessons
