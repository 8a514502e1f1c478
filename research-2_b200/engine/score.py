"""How likely a model finds given sequences of tokens: each token's log-probability behind those before it. Sequences pass through the engine's step function
in portions, as prompts do, and the head ends in the tokens' losses (`ops.token_loss`): logits of [portion, vocabulary] are at no time in memory."""

from __future__ import annotations

import numpy as np

from .replay import Replay, token_sequences


def score(model_dir, sequences, *, dtype: str = "bfloat16", device: str = "cuda:0", portion: int = 2048, block_size: int = 16) -> list[np.ndarray]:
    """For each sequence of T token ids the log-probabilities of its tokens from the second on, float32 [T - 1]: entry t is that of tokens[t + 1] behind
    tokens[: t + 1]. `portion`: rows of a step; float32 scores are the same bits whatever it is."""
    sequences = token_sequences(sequences)
    if portion < 1:
        raise ValueError(f"portion must be >= 1, got {portion}")
    longest = max((len(s) for s in sequences), default=0)
    if longest < 2:
        return [np.empty(0, dtype=np.float32) for _ in sequences]
    replay = Replay(str(model_dir), dtype, longest, block_size, device, max_live=1)
    vocab = replay.model.vocab_size
    scores = []
    for n, tokens in enumerate(sequences):
        if tokens.min() < 0 or tokens.max() >= vocab:
            raise ValueError(f"sequence {n} has tokens outside [0, {vocab})")
        parts = [np.empty(0, dtype=np.float32)]
        for begin in range(0, len(tokens) - 1, portion):   # (the last token is nobody's condition)
            rows, targets = tokens[begin: min(begin + portion, len(tokens) - 1)], tokens[begin + 1: begin + 1 + portion]
            entry = {"id": n, "tokens": rows.tolist(), "want": list(range(len(rows)))}
            parts.append(-replay.step_losses({"entries": [entry], "end": [n] if begin + portion >= len(tokens) - 1 else []}, targets))
        scores.append(np.concatenate(parts))
    return scores


__all__ = ["score"]
