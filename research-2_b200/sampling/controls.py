"""What a request may ask of its logits before a token is drawn from them: penalties for tokens that it holds already, biases of single
tokens, a grammar, and the log-probabilities beside its tokens.

A grammar is any object with two methods: `allowed()` returns which tokens may come next, as truth values [vocabulary] or as the words
that `pack_mask` makes of them, and `advance(token)` tells it which one came. A grammar follows one request; one that answers the same whatever
came says so by an attribute `stateless` that is true, and may serve any number of requests. `AllowedTokens` is the simplest: the same tokens
every time."""

from __future__ import annotations

import math
from collections.abc import Mapping
from dataclasses import dataclass

import numpy as np


def mask_words(vocab_size: int) -> int:
    return -(-vocab_size // 32)


def pack_mask(allowed: np.ndarray) -> np.ndarray:
    """Truth values [vocabulary] as int32 words: token t is bit t % 32 of word t / 32."""
    bits = np.zeros(mask_words(len(allowed)) * 32, dtype=np.uint8)
    bits[: len(allowed)] = np.asarray(allowed, dtype=bool)
    return np.packbits(bits, bitorder="little").view("<i4").astype(np.int32)


class AllowedTokens:
    """The grammar of a set of tokens: every next token is one of them."""

    stateless = True

    def __init__(self, tokens, vocab_size: int):
        tokens = np.asarray(list(tokens), dtype=np.int64)
        if len(tokens) == 0 or tokens.min() < 0 or tokens.max() >= vocab_size:
            raise ValueError(f"allowed tokens must be some of [0, {vocab_size})")
        allowed = np.zeros(vocab_size, dtype=bool)
        allowed[tokens] = True
        self._words = pack_mask(allowed)

    def allowed(self) -> np.ndarray:
        return self._words

    def advance(self, token: int) -> None:
        pass


@dataclass(frozen=True)
class Controls:
    """Tokens of the prompt and of the answer have a positive logit divided by `repetition_penalty` and another one multiplied; a token
    that stands c > 0 times in the answer then loses frequency_penalty * c + presence_penalty; `logit_bias` (token -> value, -inf forbids) is added;
    what the `grammar` forbids is -inf. `top_logprobs` n (0 to 256): `Engine.logprobs` has, for every token, its log-probability and the n
    most likely tokens with theirs, by the logits after these controls at temperature 1 (None: not kept)."""

    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Mapping[int, float] | None = None
    grammar: object | None = None
    top_logprobs: int | None = None

    def checked(self, vocab_size: int) -> "Controls":
        if not (math.isfinite(self.repetition_penalty) and self.repetition_penalty > 0):
            raise ValueError(f"repetition_penalty must be finite and > 0, got {self.repetition_penalty}")
        for name in ("presence_penalty", "frequency_penalty"):
            if not math.isfinite(getattr(self, name)):
                raise ValueError(f"{name} must be finite, got {getattr(self, name)}")
        for token, value in (self.logit_bias or {}).items():
            if not (isinstance(token, (int, np.integer)) and 0 <= token < vocab_size):
                raise ValueError(f"logit_bias names token {token!r}, the vocabulary is [0, {vocab_size})")
            if math.isnan(value) or value == math.inf:
                raise ValueError(f"logit_bias of token {token} must be a number or -inf, got {value}")
        if self.grammar is not None and not (hasattr(self.grammar, "allowed") and hasattr(self.grammar, "advance")):
            raise ValueError("a grammar has the methods allowed() and advance(token)")
        if self.top_logprobs is not None and not 0 <= self.top_logprobs <= min(256, vocab_size):
            raise ValueError(f"top_logprobs must be in [0, {min(256, vocab_size)}], got {self.top_logprobs}")
        return self

    @property
    def penalises(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    def __bool__(self) -> bool:
        """Whether anything is asked for."""
        return self.penalises or bool(self.logit_bias) or self.grammar is not None or self.top_logprobs is not None


@dataclass(frozen=True)
class TokenLogprobs:
    """A drawn token with its log-probability, and the most likely ones with theirs, from the likeliest down."""

    token: int
    logprob: float
    top: tuple[tuple[int, float], ...]


class NoTokenAllowed(RuntimeError):
    """A running request's grammar allows no token, or none that its biases do not forbid: cancel the request, or step on once its grammar does."""

    def __init__(self, req_id: int):
        super().__init__(f"request {req_id}: its grammar and its biases allow no token")
        self.req_id = req_id


__all__ = ["AllowedTokens", "Controls", "NoTokenAllowed", "TokenLogprobs", "mask_words", "pack_mask"]
