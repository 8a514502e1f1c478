"""The two ends of a token table in training, as cases that can be timed and compared.

A model's tokens come out of a table of rows and its answers are measured against the same table (or another one of its shape). Three operators stand there:

  score   the loss of given tokens, row by row, from hidden rows and the table: the logarithm of the sum of exponentials of all logits less the token's logit,
          without the logits in memory
  train   the same with the gradients of the hidden rows and of the table
  rows    the gradient of a table whose rows were looked up by tokens, many of them the same

`own` false: elementary torch operations in 32 bits. `own` true: the framework's kernels, as a program calls them.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
GPT2_VOCAB = 50257


# ---- cases --------------------------------------------------------------------------------------

def _loss(name, op, rows, width, vocab, dtype="bfloat16", padding=0, softcap=0.0, pad=0):
    """`padding`: every how-manieth row has no token to learn (0: none); `pad`: numbers between the hidden rows."""
    case = {"op": op, "rows": rows, "width": width, "vocab": vocab, "dtype": dtype, "padding": padding, "softcap": softcap, "pad": pad}
    return case if name is None else {"name": name, **case}


def _rows(name, tokens, width, vocab, dtype="bfloat16", scale=1.0, padding=0, pad=0):
    """`padding`: every how-manieth place holds no token (0: none); `pad`: numbers between the rows that come from above."""
    case = {"op": "rows", "tokens": tokens, "width": width, "vocab": vocab, "dtype": dtype, "scale": scale, "padding": padding, "pad": pad}
    return case if name is None else {"name": name, **case}


def listed() -> list[dict]:
    return [
        # how likely one token was: the table's pass alone, latency
        _loss("score one row", "score", 1, 768, GPT2_VOCAB),
        # a prompt of odd length scored in the 32-bit path
        _loss("score 100 float32 rows", "score", 100, 768, GPT2_VOCAB, "float32"),
        # a corpus scored two whole contexts at a time
        _loss("score 2 x 1,024 rows", "score", 2048, 768, GPT2_VOCAB, padding=1024),
        # GPT-2 1.5B's width, a ragged batch with padding, rows of a wider buffer
        _loss("score 1,000 wide rows", "score", 1000, 1600, GPT2_VOCAB, padding=9, pad=8),
        # a small student of odd sizes on a short batch: latency
        _loss("train sixteen rows", "train", 16, 100, 1031, "float32"),
        # a student in 32 bits, half a context
        _loss("train 512 float32 rows", "train", 512, 768, GPT2_VOCAB, "float32", padding=16),
        # a step of training in bfloat16, four contexts
        _loss("train 4,096 rows", "train", 4096, 768, GPT2_VOCAB, padding=16),
        # a wide model with a wide table of odd size and capped logits, a ragged number of rows
        _loss("train 2,047 wide rows", "train", 2047, 1600, 128001, padding=16, softcap=30.0),
        # a short sequence of a small student: latency
        _rows("rows of sixteen tokens", 16, 100, 1031, "float32"),
        # one context, a table of which most rows get nothing
        _rows("rows of 1,024 tokens", 1024, 768, GPT2_VOCAB, "float32", padding=16),
        # a step of training in bfloat16, with a scaled table
        _rows("rows of 4 x 1,024 tokens", 4096, 768, GPT2_VOCAB, scale=8.0, padding=16),
        # a large batch of a wide model: some tokens stand in it thousands of times
        _rows("rows of 32 x 1,024 tokens", 32768, 1600, GPT2_VOCAB),
    ]


MOST_PRODUCTS = 2047 * 1600 * 128001       # of a drawn training step in bfloat16
MOST_NUMBERS = (32768 + GPT2_VOCAB) * 1600   # of a drawn table with the rows from above


def draw(rng) -> dict:
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op, dtype, pad = rng.choice(["score", "train", "rows"]), rng.choice(["bfloat16", "bfloat16", "float32"]), rng.choice([0, 0, 0, 1, 8, 40])
    vocab, width = rng.choice([GPT2_VOCAB, spread(300, 160000)]), rng.choice([768, 1024, spread(33, 1600)])
    padding = rng.choice([0, 3, 16])
    if op == "rows":
        tokens = max(1, min(spread(1, 40000), MOST_NUMBERS // width - vocab))
        vocab = min(vocab, MOST_NUMBERS // width - tokens)
        return _rows(None, tokens, width, vocab, dtype, rng.choice([1.0, round(rng.uniform(0.1, 30.0), 3)]), padding, pad)
    rows = max(1, min(spread(1, 5000), MOST_PRODUCTS // (width * vocab * (6 if dtype == "float32" else 1))))
    return _loss(None, op, rows, width, vocab, dtype, padding, rng.choice([0.0, 0.0, 30.0, round(rng.uniform(5.0, 60.0), 2)]), pad)


# ---- what a program has in hand -----------------------------------------------------------------

def _strided(values: torch.Tensor, dtype: str, pad: int) -> torch.Tensor:
    """The rows as a buffer whose rows have `pad` places more than they use."""
    rows, width = values.shape
    buffer = torch.zeros(rows, width + pad, dtype=getattr(torch, dtype), device=DEV)
    buffer[:, :width] = values
    return buffer[:, :width]


def _tokens(n: int, vocab: int, gen: torch.Generator) -> torch.Tensor:
    """Tokens as text has them: few of them often (one of ten places is the commonest's), most of them seldom."""
    draws = torch.rand(n, generator=gen, device=DEV)
    tokens = (vocab * draws ** 3).long().clamp_(max=vocab - 1)
    return torch.where(torch.rand(n, generator=gen, device=DEV) < 0.1, 13 % vocab, tokens).to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    state = dict(case)
    width, vocab, dtype = case["width"], case["vocab"], case["dtype"]
    if case["op"] == "rows":
        n = case["tokens"]
        ids = _tokens(n, vocab, gen)
        if case["padding"]:
            ids[case["padding"] - 1::case["padding"]] = -1
        state["ids"] = ids
        state["above"] = _strided(1e-3 * torch.randn(n, width, generator=gen, device=DEV), dtype, case["pad"])
        return state
    rows = case["rows"]
    # a table whose logits have a deviation of two, and hidden rows of which some know their token and others do not
    table = torch.randn(vocab, width, generator=gen, device=DEV) * (2.0 / math.sqrt(width))
    targets = _tokens(rows, vocab, gen)
    know = 2.5 * torch.rand(rows, 1, generator=gen, device=DEV)
    hidden = torch.randn(rows, width, generator=gen, device=DEV) + know * table[targets.long()]
    weight = (0.5 + torch.rand(rows, generator=gen, device=DEV)) / rows
    if case["padding"]:
        targets[case["padding"] - 1::case["padding"]] = -1
    state["table"] = table.to(getattr(torch, dtype))
    state["hidden"] = _strided(hidden, dtype, case["pad"])
    state["targets"] = targets
    state["weight"] = weight if case["op"] == "train" else None
    return state


# ---- one pass -----------------------------------------------------------------------------------

def run(state: dict):
    if own:
        from research_2_b200.kernels import ops

        if state["op"] == "rows":
            return ops.token_rows_gradient(state["ids"], state["above"], state["vocab"], scale=state["scale"])
        loss, log_sum = ops.token_loss(state["hidden"], state["table"], state["targets"], weight=state["weight"], softcap=state["softcap"])
        if state["op"] == "score":
            return loss, log_sum
        d_hidden, d_table = ops.token_loss_gradient(state["hidden"], state["table"], state["targets"], log_sum, weight=state["weight"],
                                                    softcap=state["softcap"])
        return loss, d_hidden, d_table
    return _plain_rows(state) if state["op"] == "rows" else _plain_loss(state)


def _plain_loss(s: dict):
    x, w, targets, softcap = s["hidden"].float(), s["table"].float(), s["targets"], s["softcap"]
    z = x @ w.t()
    if softcap > 0:
        z = softcap * torch.tanh(z / softcap)
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    log_sum = (top + torch.log(total))[:, 0]
    held = (targets >= 0) & (targets < s["vocab"])
    at = targets.clamp(0, s["vocab"] - 1).long()[:, None]
    loss = torch.where(held, log_sum - torch.gather(z, 1, at)[:, 0], 0.0)
    if s["op"] == "score":
        return loss, log_sum
    factor = torch.where(held, s["weight"], 0.0)[:, None]
    dz = (e / total).scatter_add_(1, at, torch.full_like(total, -1.0)) * factor
    if softcap > 0:
        dz = dz * (1.0 - (z / softcap) ** 2)
    return loss * s["weight"], (dz @ w).to(s["hidden"].dtype), (dz.t() @ x).to(s["table"].dtype)


def _plain_rows(s: dict) -> torch.Tensor:
    ids = s["ids"].long()
    held = (ids >= 0) & (ids < s["vocab"])
    above = s["above"].float() * s["scale"]
    # one row more than the table's, for places without a token
    table = torch.zeros(s["vocab"] + 1, s["width"], device=above.device)
    table.index_add_(0, torch.where(held, ids, s["vocab"]), above)
    return table[:-1].to(s["above"].dtype)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case: dict) -> dict:
    width, vocab, size = case["width"], case["vocab"], 4 if case["dtype"] == "float32" else 2
    n = case["tokens"] if case["op"] == "rows" else case["rows"]
    counted = n - (n // case["padding"] if case["padding"] else 0)   # a place without a token need not be read
    if case["op"] == "rows":
        return {"bytes": 4 * n + counted * width * size + vocab * width * size, "flops": counted * width}
    read = (n if case["op"] == "score" else counted) * width * size + vocab * width * size + 4 * n
    if case["op"] == "score":
        return {"bytes": read + 8 * n, "flops": 2 * n * width * vocab}
    return {"bytes": read + 8 * n + n * width * size + vocab * width * size, "flops": 6 * counted * width * vocab}


# ---- the same from the definitions, in 64 bits --------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "rows":
        return _exact_rows(s)
    w, cap, train = s["table"].double(), float(s["softcap"]), case["op"] == "train"
    losses, log_sums, d_hidden, d_table = [], [], [], torch.zeros_like(w) if train else None
    step = max(1, 60_000_000 // case["vocab"])
    for begin in range(0, case["rows"], step):
        x = s["hidden"][begin: begin + step].double()
        y = s["targets"][begin: begin + step].long()
        u = torch.matmul(x, w.T)
        z = cap * torch.tanh(u / cap) if cap else u
        log_q = torch.log_softmax(z, dim=1)
        log_sums.append(torch.logsumexp(z, dim=1))
        learns = (0 <= y) & (y < case["vocab"])
        which = torch.nonzero(learns)[:, 0]
        loss = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
        loss[which] = -log_q[which, y[which]]
        if train:
            weight = s["weight"][begin: begin + step].double()
            loss = loss * weight
            g = torch.exp(log_q)
            g[which, y[which]] -= 1.0
            g = g * (weight * learns)[:, None]
            if cap:
                g = g / torch.cosh(u / cap) ** 2
            d_hidden.append(torch.matmul(g, w))
            d_table += torch.matmul(g.T, x)
        losses.append(loss)
    if train:
        return torch.cat(losses), torch.cat(d_hidden), d_table
    return torch.cat(losses), torch.cat(log_sums)


def _exact_rows(s: dict) -> torch.Tensor:
    held = torch.nonzero((s["ids"] >= 0) & (s["ids"] < s["vocab"]))[:, 0]
    order = held[torch.argsort(s["ids"][held], stable=True)]
    rows = float(s["scale"]) * s["above"][order].double()
    tokens, counts = torch.unique_consecutive(s["ids"][order].long(), return_counts=True)
    out = torch.zeros(s["vocab"], s["width"], dtype=torch.float64, device=rows.device)
    # one token after the other by places within its run, the longest run's number of turns at most
    ends = torch.cumsum(counts, 0)
    if rows.shape[0] * rows.shape[1] < 4_000_000:
        for token, end, count in zip(tokens.tolist(), ends.tolist(), counts.tolist()):
            out[token] = rows[end - count: end].sum(dim=0)
        return out
    sums = torch.cumsum(rows, dim=0)   # (64 bits bear the difference of two running sums)
    before = torch.where((ends > counts)[:, None], sums[(ends - counts - 1).clamp(min=0)], 0.0)
    out[tokens] = sums[ends - 1] - before
    return out
