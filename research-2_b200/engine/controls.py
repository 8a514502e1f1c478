"""Steps whose requests ask something of their logits (`sampling.controls`): the pass runs as it always does, and between its logits and
the draw stand one launch that adjusts them, in place, and where log-probabilities are asked for one that takes the largest. What requests
hold is kept on the device, a row of tokens per request slot, from the step's own rows."""

from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

from ..kernels import ops
from ..sampling.controls import Controls, NoTokenAllowed, TokenLogprobs, mask_words, pack_mask


@dataclass
class _Request:
    controls: Controls
    n_prompt: int
    bias_ids: np.ndarray
    bias_values: np.ndarray
    mask: np.ndarray | None = None      # words, what the grammar allows next
    logprobs: list[TokenLogprobs] = field(default_factory=list)
    not_forbidden: np.ndarray | None = None   # words, what biases of -inf leave (None: there are none)
    failure: Exception | None = None          # of its grammar, when it was told a token or asked after it

    def nothing_left(self) -> bool:
        """Whether no token may be drawn."""
        if self.not_forbidden is None:
            return self.mask is not None and not self.mask.any()
        left = self.not_forbidden if self.mask is None else self.mask & self.not_forbidden
        return not left.any()


def allowed_words(grammar, vocab_size: int) -> np.ndarray:
    """What a grammar allows next, as int32 words; bits beyond the vocabulary are cleared."""
    words, allowed = mask_words(vocab_size), np.asarray(grammar.allowed())
    if allowed.dtype == bool:
        if allowed.shape != (vocab_size,):
            raise ValueError(f"a grammar's allowed() must have {vocab_size} truth values, got shape {allowed.shape}")
        return pack_mask(allowed)
    if allowed.dtype not in (np.int32, np.uint32) or allowed.shape != (words,):
        raise ValueError(f"a grammar's allowed() must be {vocab_size} truth values or {words} words of 32 bits, got {allowed.dtype} {allowed.shape}")
    out = allowed.view(np.int32).copy() if allowed.flags.c_contiguous else np.ascontiguousarray(allowed).view(np.int32)
    if vocab_size % 32:
        out[-1] &= np.int32((1 << (vocab_size % 32)) - 1)
    return out


def pack_rows(rows: list[_Request | None], vocab_size: int) -> tuple[np.ndarray, dict[str, tuple[int, int, type]]]:
    """What adjusting needs of a step's rows besides their histories, as one int32 array and where each part lies in it: (first, count,
    type). A row of None, or one that does not ask for a part, is neutral."""
    n, words = len(rows), mask_words(vocab_size)
    n_biases = sum(len(r.bias_ids) for r in rows if r is not None)
    n_masks = sum(r is not None and r.mask is not None for r in rows)
    parts, at = {}, 0
    for name, count, kind in (("prompt_lengths", n, np.int32), ("repetition", n, np.float32), ("presence", n, np.float32), ("frequency", n, np.float32),
                              ("mask_rows", n, np.int32), ("bias_start", n + 1, np.int32), ("bias_ids", n_biases, np.int32),
                              ("bias_values", n_biases, np.float32), ("mask", n_masks * words, np.int32)):
        parts[name] = (at, count, kind)
        at += -(-max(count, 1) // 4) * 4   # parts start on 16-byte boundaries
    out = np.zeros(at, dtype=np.int32)

    def part(name: str) -> np.ndarray:
        first, count, kind = parts[name]
        return out[first: first + count].view(kind)

    prompt_lengths, repetition, presence, frequency = (part(name) for name in ("prompt_lengths", "repetition", "presence", "frequency"))
    mask_rows, bias_start, bias_ids, bias_values, mask = (part(name) for name in ("mask_rows", "bias_start", "bias_ids", "bias_values", "mask"))
    repetition[:] = 1.0
    mask_rows[:] = -1
    bias, which = 0, 0
    for i, r in enumerate(rows):
        if r is not None:
            prompt_lengths[i] = r.n_prompt
            repetition[i], presence[i], frequency[i] = r.controls.repetition_penalty, r.controls.presence_penalty, r.controls.frequency_penalty
            bias_ids[bias: bias + len(r.bias_ids)] = r.bias_ids
            bias_values[bias: bias + len(r.bias_ids)] = r.bias_values
            bias += len(r.bias_ids)
            if r.mask is not None:
                mask_rows[i] = which
                mask[which * words: (which + 1) * words] = r.mask
                which += 1
        bias_start[i + 1] = bias
    return out, parts


class StepControls:
    """The controlled requests of one engine, by request id."""

    def __init__(self, step_fn, max_requests: int, max_seq_len: int, vocab_size: int):
        self.step_fn, self.vocab_size = step_fn, vocab_size
        self.shape = (max_requests, max_seq_len)
        self.requests: dict[int, _Request] = {}
        self.ended: dict[int, _Request] = {}      # their log-probabilities are kept until the id is given again
        self._history: torch.Tensor | None = None
        self._done: torch.cuda.Event | None = None

    def asked(self, controls: Controls, n_prompt: int) -> _Request:
        """What a request will ask of its rows; its grammar is asked what may come first, so what is wrong with it shows here, before there is a request."""
        shared = controls.grammar is not None and any(r.controls.grammar is controls.grammar for r in self.requests.values())
        if shared and not getattr(controls.grammar, "stateless", False):
            raise ValueError("this grammar follows another request: give each request one of its own (or let it say that it is `stateless`)")
        biases = sorted((controls.logit_bias or {}).items())
        request = _Request(controls, n_prompt, np.array([t for t, _ in biases], dtype=np.int32), np.array([v for _, v in biases], dtype=np.float32))
        forbidden = request.bias_ids[request.bias_values == -np.inf]
        if len(forbidden):
            left = np.ones(self.vocab_size, dtype=bool)
            left[forbidden] = False
            request.not_forbidden = pack_mask(left)
        if controls.grammar is not None:
            request.mask = allowed_words(controls.grammar, self.vocab_size)
        return request

    def add(self, rid: int, request: _Request) -> None:
        self.requests[rid] = request

    def forget(self, rid: int, keep: bool = False) -> None:
        request = self.requests.pop(rid, None)
        self.ended.pop(rid, None)
        if keep and request is not None:
            self.ended[rid] = request

    def logprobs(self, rid: int) -> list[TokenLogprobs]:
        request = self.requests.get(rid) or self.ended.get(rid)
        if request is None:
            raise KeyError(f"no request {rid} with controls")
        return list(request.logprobs)

    def check(self, is_live) -> None:
        """Raises NoTokenAllowed where a live request's grammar allows nothing, or nothing that its biases do not forbid (the grammar is asked
        again each time: it may have been told more), and what its grammar raised when it was told a token."""
        for rid, request in self.requests.items():
            if request.failure is not None and is_live(rid):
                raise request.failure
            if request.nothing_left() and is_live(rid):
                if request.mask is not None:
                    request.mask = allowed_words(request.controls.grammar, self.vocab_size)
                if request.nothing_left():
                    raise NoTokenAllowed(rid)

    def concerns(self, plan) -> bool:
        return any(int(r) in self.requests for r in plan.req)

    @torch.no_grad()
    def step(self, batch, plan) -> np.ndarray:
        """The pass of a batch with controlled requests: one token per entry, on the host. What the requests' grammars and records learn
        of it is told by `committed`."""
        step_fn, n = self.step_fn, plan.n_entries
        rows = [self.requests.get(int(rid)) if emits else None for rid, emits in zip(plan.req, plan.emits)]
        with torch.cuda.device(step_fn.device):
            logits, ctx = step_fn.logits_and_context(batch)
            if self._history is None:
                self._history = torch.zeros(self.shape, dtype=torch.int32, device=step_fn.device)
            ops.keep_tokens(self._history, ctx.input_ids, ctx.positions, ctx.row_entry, ctx.state_slot)
            packed, parts = pack_rows(rows, self.vocab_size)
            dev = torch.from_numpy(packed).pin_memory().to(step_fn.device, non_blocking=True)

            def part(name: str) -> torch.Tensor | None:
                first, count, kind = parts[name]
                view = dev[first: first + count]
                return view.view(torch.float32) if kind is np.float32 else view

            arguments = {}
            if any(r is not None and r.controls.penalises for r in rows):
                arguments.update(history=self._history, slots=ctx.state_slot, lengths=ctx.seq_lens, prompt_lengths=part("prompt_lengths"),
                                 repetition=part("repetition"), presence=part("presence"), frequency=part("frequency"))
            if parts["bias_ids"][1]:
                arguments.update(bias_start=part("bias_start"), bias_ids=part("bias_ids"), bias_values=part("bias_values"))
            if parts["mask"][1]:
                arguments.update(mask=part("mask").view(-1, mask_words(self.vocab_size)), mask_rows=part("mask_rows"))
            if arguments:
                ops.adjust_logits(logits, **arguments, out=logits)
            tokens = step_fn.sample(logits, ctx)[:n]
            asked = [r.controls.top_logprobs for r in rows if r is not None and r.controls.top_logprobs is not None]
            self._top = None
            if asked:
                values, ids, log_sum = ops.top_logits(logits, max(1, max(asked)))
                chosen = torch.gather(logits, 1, tokens.long()[:, None])
                self._top = [t.cpu().numpy() for t in (values, ids, log_sum, chosen[:, 0])]
            if step_fn.order is not None:   # (these launches belong to the pass: one on another stream waits for them too)
                if self._done is None:
                    self._done = torch.cuda.Event()
                step_fn.order.end(self._done)
            out = tokens.cpu().numpy()
        ops.raise_on_device_error(step_fn.device)
        return out

    def committed(self, plan, tokens: np.ndarray) -> None:
        """After the step's commit: grammars go on, log-probabilities are written down. What a grammar raises is raised when all requests have
        been seen to (and again before each step, while its request lives: nobody knows what it allows)."""
        failure = None
        for e, (rid, emits) in enumerate(zip(plan.req, plan.emits)):
            request = self.requests.get(int(rid)) if emits else None
            if request is None:
                continue
            n_top = request.controls.top_logprobs
            if n_top is not None:
                values, ids, log_sum, chosen = (a[e] for a in self._top)
                top = tuple((int(i), float(v - log_sum)) for v, i in zip(values[:n_top], ids[:n_top]))
                request.logprobs.append(TokenLogprobs(int(tokens[e]), float(chosen - log_sum), top))
            if request.controls.grammar is not None:
                try:
                    request.controls.grammar.advance(int(tokens[e]))
                    request.mask = allowed_words(request.controls.grammar, self.vocab_size)
                except Exception as raised:  # noqa: BLE001
                    request.failure = raised
                    failure = failure or raised
        if failure is not None:
            raise failure
