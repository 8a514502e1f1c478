"""The operators on rows of logits, as cases that can be timed and compared.

What a model answers with is made from its logits, and so is what another model learns from it. Three operators stand there:

  adjust    penalties for tokens that a request holds already, biases of single tokens and a grammar's mask, laid on a step's logits before a
            token is drawn from them
  top       the k largest logits of every row with their tokens, in order, and the logarithm of the whole row's sum of exponentials: the
            log-probabilities beside an answer, and what a teacher writes down of a prompt's rows
  distill   a student's loss against a teacher's top logits, row by row, and the gradient with respect to the student's logits

`own` false: elementary torch operations in 32 bits. `own` true: the framework's kernels, as a program calls them.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
GPT2_VOCAB = 50257


# ---- cases --------------------------------------------------------------------------------------

def _adjust(name, rows, vocab, dtype="float32", history=0, biases=0, masks=0, pad=0):
    """`history`: the most tokens that a row's request holds; `biases`: tokens of a row with a bias; `masks`: every how-manieth row has a grammar (0: none)."""
    case = {"op": "adjust", "rows": rows, "vocab": vocab, "dtype": dtype, "history": history, "biases": biases, "masks": masks, "pad": pad}
    return case if name is None else {"name": name, **case}


def _top(name, rows, vocab, k, dtype="float32", temperature=1.0, pad=0):
    case = {"op": "top", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "temperature": temperature, "pad": pad}
    return case if name is None else {"name": name, **case}


def _distill(name, rows, vocab, k, dtype="float32", temperature=1.0, tail=True, gradient=True, padding=0, pad=0):
    """`tail`: the teacher's other tokens count as one outcome; `padding`: every how-manieth row has the weight 0 (0: none)."""
    case = {"op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "temperature": temperature, "tail": tail, "gradient": gradient,
            "padding": padding, "pad": pad}
    return case if name is None else {"name": name, **case}


def listed() -> list[dict]:
    return [
        # one request that decodes with a repetition penalty and a short history: latency alone
        _adjust("adjust one row", 1, GPT2_VOCAB, history=24, biases=2),
        # a small service: eight requests, every other one held to a grammar
        _adjust("adjust eight rows", 8, GPT2_VOCAB, history=600, biases=8, masks=2),
        # the benchmark's widest decode batch, long histories, biases on the tokens that a user lists
        _adjust("adjust sixty-four rows", 64, GPT2_VOCAB, history=1000, biases=64, masks=2),
        # as many requests as an engine batches by default at most, a wide table of odd size, bfloat16 logits in a padded buffer
        _adjust("adjust 256 bfloat16 rows", 256, 128001, "bfloat16", history=4000, biases=300, masks=1, pad=7),
        # log-probabilities beside one request's answer
        _top("top five of one row", 1, GPT2_VOCAB, 5),
        # the same for a full decode batch
        _top("top twenty of sixty-four rows", 64, GPT2_VOCAB, 20),
        # a teacher writes down a prompt of two whole contexts
        _top("teacher of 2 x 1,024 rows", 2048, GPT2_VOCAB, 64, temperature=2.0),
        # a teacher with a wide table whose logits are bfloat16 (equal values abound)
        _top("teacher of 1,000 bfloat16 rows", 1000, 128001, 128, "bfloat16", pad=7),
        # a small student's short batch: latency
        _distill("distill sixteen rows", 16, 1031, 8),
        # a student at GPT-2's table, one context, the rest of the teacher's mass as one outcome
        _distill("distill 1,024 rows", 1024, GPT2_VOCAB, 64, temperature=2.0, padding=16),
        # a step of training in bfloat16: four contexts, the teacher's mass spread over its top tokens alone
        _distill("distill 4,096 bfloat16 rows", 4096, GPT2_VOCAB, 32, "bfloat16", tail=False, padding=9),
        # a validation pass: losses without a gradient, a wide table of odd size
        _distill("losses of 2,047 rows", 2047, 128001, 100, gradient=False, padding=16, pad=3),
    ]


MOST_NUMBERS = 4096 * GPT2_VOCAB   # of a drawn case's logits


def draw(rng) -> dict:
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op, dtype, pad = rng.choice(["adjust", "top", "distill"]), rng.choice(["float32", "float32", "bfloat16"]), rng.choice([0, 0, 0, 1, 5, 8, 64])
    vocab = rng.choice([GPT2_VOCAB, spread(300, 160000)])
    if op == "adjust":
        rows = min(spread(1, 300), MOST_NUMBERS // vocab)
        return _adjust(None, rows, vocab, dtype, rng.choice([0, spread(1, 6000)]), rng.choice([0, spread(1, min(300, vocab))]), rng.choice([0, 1, 2, 5]), pad)
    rows = min(spread(1, 4096), MOST_NUMBERS // (vocab if op == "distill" else 4 * vocab))
    k, temperature = spread(1, 128), rng.choice([1.0, round(rng.uniform(0.5, 3.0), 3)])
    if op == "top":
        return _top(None, rows, vocab, k, dtype, temperature, pad)
    return _distill(None, rows, vocab, k, dtype, temperature, rng.random() < 0.6, rng.random() < 0.75, rng.choice([0, 3, 16]), pad)


# ---- what a program has in hand -----------------------------------------------------------------

def _rows(values: torch.Tensor, dtype: str, pad: int) -> torch.Tensor:
    """The rows as a buffer whose rows have `pad` places more than they use."""
    rows, vocab = values.shape
    buffer = torch.zeros(rows, vocab + pad, dtype=getattr(torch, dtype), device=DEV)
    buffer[:, :vocab] = values
    return buffer[:, :vocab]


def _random_logits(rows: int, vocab: int, gen: torch.Generator) -> torch.Tensor:
    """Logits as a language model has them: a few tokens far above a crowd that falls with the token's rank, ranks in no order of the tokens."""
    order = torch.randperm(vocab, generator=gen, device=DEV)
    crowd = -0.8 * torch.log1p(order.float())
    return 2.0 * torch.randn(rows, vocab, generator=gen, device=DEV) + crowd


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rows, vocab, dtype, pad = case["rows"], case["vocab"], case["dtype"], case["pad"]
    state = dict(case)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    if case["op"] == "adjust":
        state["logits"] = _rows(_random_logits(rows, vocab, gen) + 3.0, dtype, pad)
        most = case["history"]
        state["history"] = None
        if most:
            # one place more than there are rows, in another order: requests come and go
            tokens = (vocab * uniform(rows + 1, most) ** 3).to(torch.int32).clamp_(max=vocab - 1)
            state["history"] = tokens
            state["slots"] = torch.randperm(rows + 1, generator=gen, device=DEV)[:rows].to(torch.int32)
            state["lengths"] = (most * (0.5 + 0.5 * uniform(rows))).round().to(torch.int32)
            state["prompt_lengths"] = (state["lengths"] * uniform(rows)).to(torch.int32)
            state["repetition"] = 1.0 + 0.3 * uniform(rows)
            state["presence"] = 0.6 * uniform(rows)
            state["frequency"] = 0.4 * uniform(rows)
        n = case["biases"]
        state["bias_start"] = None
        if n:
            counts = torch.full((rows,), n, device=DEV)
            counts[1::3] = n // 2    # requests list as many as they like, some none
            counts[2::7] = 0
            start = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
            start[1:] = counts.cumsum(0)
            total = int(start[-1])
            step = max(1, vocab // n)    # a token stands once in a row
            places = torch.arange(total, device=DEV) - torch.repeat_interleave(start[:-1].long(), counts)
            state["bias_start"] = start
            state["bias_ids"] = (places * step + (uniform(total) * step).long()).clamp_(max=vocab - 1).to(torch.int32)
            state["bias_values"] = 4.0 * uniform(total) - 2.0
        state["mask"] = None
        if case["masks"]:
            which = torch.arange(rows, device=DEV) % case["masks"] == 0
            n_masks = int(which.sum())
            words = (vocab + 31) // 32
            dense = torch.randint(-2**31, 2**31, (n_masks, words), generator=gen, device=DEV, dtype=torch.int64)
            sparse = dense & torch.randint(-2**31, 2**31, (n_masks, words), generator=gen, device=DEV, dtype=torch.int64) & (dense >> 7) & (dense >> 13) & (dense >> 5)
            few = torch.arange(n_masks, device=DEV)[:, None] % 3 != 1    # most grammars leave few tokens, some half of them
            state["mask"] = torch.where(few, sparse, dense).to(torch.int32)
            state["mask_rows"] = torch.where(which, which.long().cumsum(0) - 1, -1).to(torch.int32)
        return state
    teacher = _random_logits(rows, vocab, gen)
    if case["op"] == "top":
        state["logits"] = _rows(teacher, dtype, pad)
        return state
    k = min(case["k"], vocab)
    student = teacher + 1.5 * torch.randn(rows, vocab, generator=gen, device=DEV)
    values, ids = torch.topk(teacher, k, dim=1)
    fewer = (uniform(rows, 1) < 0.1) & (torch.arange(k, device=DEV) >= k - k // 4)   # some rows hold fewer
    state["ids"] = torch.where(fewer, -1, ids).to(torch.int32)
    state["teacher"] = values
    state["log_sum"] = torch.logsumexp(teacher / case["temperature"], dim=1) if case["tail"] else None
    state["logits"] = _rows(student, dtype, pad)
    weight = 0.5 + uniform(rows)
    if case["padding"]:
        weight[case["padding"] - 1::case["padding"]] = 0.0
    state["weight"] = weight
    return state


# ---- one pass -----------------------------------------------------------------------------------

def run(state: dict):
    if own:
        from research_2_b200.kernels import ops

        if state["op"] == "adjust":
            return ops.adjust_logits(state["logits"], history=state["history"], slots=state.get("slots"), lengths=state.get("lengths"),
                                     prompt_lengths=state.get("prompt_lengths"), repetition=state.get("repetition"), presence=state.get("presence"),
                                     frequency=state.get("frequency"), bias_start=state["bias_start"], bias_ids=state.get("bias_ids"),
                                     bias_values=state.get("bias_values"), mask=state["mask"], mask_rows=state.get("mask_rows"))
        if state["op"] == "top":
            return ops.top_logits(state["logits"], min(state["k"], state["vocab"]), temperature=state["temperature"])
        loss, gradient = ops.distill_loss(state["logits"], state["ids"], state["teacher"], log_sum=state["log_sum"], temperature=state["temperature"],
                                          weight=state["weight"], gradient=state["gradient"])
        return (loss, gradient) if state["gradient"] else loss
    return {"adjust": _plain_adjust, "top": _plain_top, "distill": _plain_distill}[state["op"]](state)


def _plain_adjust(s: dict) -> torch.Tensor:
    x = s["logits"].float()
    rows, vocab = x.shape
    if s["history"] is not None:
        held = s["history"][s["slots"].long()].long()
        at = torch.arange(held.shape[1], device=x.device)
        present = at < s["lengths"][:, None]
        drawn = present & (at >= s["prompt_lengths"][:, None])
        seen = torch.zeros_like(x).scatter_add_(1, held, present.float()) > 0
        count = torch.zeros_like(x).scatter_add_(1, held, drawn.float())
        repetition = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
        x = x - (s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0))
    if s["bias_start"] is not None:
        n = torch.arange(s["bias_ids"].shape[0], device=x.device, dtype=torch.int32)
        row = torch.searchsorted(s["bias_start"], n, right=True) - 1
        x = x + torch.zeros_like(x).index_put_((row, s["bias_ids"].long()), s["bias_values"])
    if s["mask"] is not None:
        token = torch.arange(vocab, device=x.device)
        words = s["mask"][s["mask_rows"].clamp(min=0).long()]
        forbidden = ((words[:, token // 32] >> (token % 32)) & 1) == 0
        x = torch.where(forbidden & (s["mask_rows"] >= 0)[:, None], -math.inf, x)
    return x.to(s["logits"].dtype)


def _plain_top(s: dict):
    x = s["logits"].float()
    values, ids = torch.sort(x, dim=1, descending=True, stable=True)
    k = min(s["k"], s["vocab"])
    top = values[:, :1] / s["temperature"]
    log_sum = top[:, 0] + torch.log(torch.sum(torch.exp(x / s["temperature"] - top), dim=1))
    return values[:, :k].contiguous(), ids[:, :k].to(torch.int32), log_sum


def _plain_distill(s: dict):
    z = s["logits"].float() / s["temperature"]
    m = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(dim=1, keepdim=True)
    held = s["ids"] >= 0
    ids = s["ids"].clamp(min=0).long()
    t = torch.where(held, s["teacher"] / s["temperature"], -math.inf)
    if s["log_sum"] is None:
        t_max = t.amax(dim=1, keepdim=True)
        log_p = t - t_max - torch.log(torch.exp(t - t_max).sum(dim=1, keepdim=True))
    else:
        log_p = t - s["log_sum"][:, None]
    p = torch.exp(log_p)
    log_q = torch.gather(z - m, 1, ids) - torch.log(total)
    d = log_p - log_q
    mass = p.sum(dim=1, keepdim=True)
    if s["log_sum"] is None:
        kl = torch.where(p > 0, p * d, 0.0).sum(dim=1)
        factor = mass
    else:
        # sum of p log(p / q) over outcomes that are whole on both sides, as terms p log(p / q) - p + q, none of which is negative
        q = torch.where(held, torch.exp(log_q), 0.0)
        others = torch.ones_like(z).scatter_add_(1, ids, -held.float())
        rest = (e * others).sum(dim=1, keepdim=True) / total
        rest_p = torch.where(rest > 0, (1.0 - mass).clamp(min=0.0), 0.0)
        rest_d = torch.log(rest_p) - torch.log(rest)
        kl = torch.where(held & (p > 0), p * (d + torch.expm1(-d)), q).sum(dim=1)
        kl = kl + torch.where(rest_p > 0, rest_p * (rest_d + torch.expm1(-rest_d)), torch.where(rest > 0, rest, mass - 1.0))[:, 0]
        outside = torch.where(rest_p > 0, (mass - q.sum(dim=1, keepdim=True)) / rest, mass)
        factor = torch.where(others > 0, outside, torch.where(rest_p > 0, 1.0, mass))
    weight = s["weight"]
    loss = torch.where(weight == 0, 0.0, weight * (s["temperature"] ** 2) * kl)
    if not s["gradient"]:
        return loss
    gradient = (e / total * factor).scatter_add_(1, ids, torch.where(held, -p, 0.0))
    gradient = torch.where(weight[:, None] == 0, 0.0, gradient * (weight * s["temperature"])[:, None])
    return loss, gradient.to(s["logits"].dtype)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case: dict) -> dict:
    rows, vocab, size = case["rows"], case["vocab"], 4 if case["dtype"] == "float32" else 2
    numbers = rows * vocab
    if case["op"] == "adjust":
        masked = -(-rows // case["masks"]) if case["masks"] else 0
        held = 0.75 * case["history"] * rows
        return {"bytes": 2 * numbers * size + masked * vocab / 8 + 4 * held + 6 * case["biases"] * rows + 28 * rows, "flops": 4 * held + case["biases"] * rows}
    k = min(case["k"], vocab)
    if case["op"] == "top":
        return {"bytes": numbers * size + 8 * k * rows + 4 * rows, "flops": 4 * numbers}
    counted = rows - (rows // case["padding"] if case["padding"] else 0)   # a row that weighs nothing need not be read
    read, written = counted * vocab * size + 8 * k * counted + 8 * rows, 4 * rows + (numbers * size if case["gradient"] else 0)
    return {"bytes": read + written, "flops": (7 if case["gradient"] else 4) * counted * vocab}


# ---- the same from the definitions, in 64 bits --------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    parts = []
    rows = case["rows"]
    step = max(1, 40_000_000 // case["vocab"])
    for begin in range(0, rows, step):
        parts.append(_EXACT[case["op"]](s, slice(begin, min(rows, begin + step))))
    if isinstance(parts[0], tuple):
        return tuple(None if column[0] is None else torch.cat(column) for column in zip(*parts))
    return torch.cat(parts)


def _exact_adjust(s: dict, part: slice) -> torch.Tensor:
    x = s["logits"][part].double()
    n = x.shape[0]
    for i in range(n):
        row = part.start + i
        if s["history"] is not None:
            length, prompt = int(s["lengths"][row]), int(s["prompt_lengths"][row])
            held = s["history"][int(s["slots"][row]), :length].long()
            rho = s["repetition"][row].double()
            every = held.unique()
            old = x[i, every]
            x[i, every] = torch.where(old > 0, old / rho, old * rho)
            drawn, count = held[min(prompt, length):].unique(return_counts=True)
            x[i, drawn] -= s["presence"][row].double() + count.double() * s["frequency"][row].double()
        if s["bias_start"] is not None:
            a, b = int(s["bias_start"][row]), int(s["bias_start"][row + 1])
            x[i, s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        if s["mask"] is not None and int(s["mask_rows"][row]) >= 0:
            words = s["mask"][int(s["mask_rows"][row])]
            bits = (words[:, None].long() >> torch.arange(32, device=x.device)) % 2 != 0
            x[i, ~bits.reshape(-1)[: x.shape[1]]] = -math.inf
    return x


def _exact_top(s: dict, part: slice):
    x = s["logits"][part].double()
    k = min(s["k"], s["vocab"])
    # (values that stand k times or more at the edge: the composite of value and token orders them)
    place = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
    return torch.gather(x, 1, place), place.to(torch.int32), torch.logsumexp(x / float(s["temperature"]), dim=1)


def _exact_distill(s: dict, part: slice):
    x, tau = s["logits"][part].double(), float(s["temperature"])
    ids, held = s["ids"][part].long(), s["ids"][part] >= 0
    t = s["teacher"][part].double() / tau
    weight = s["weight"][part].double()
    # the teacher's distribution over the table: its top tokens, and one more place for all others
    target = torch.zeros(x.shape[0], x.shape[1] + 1, dtype=torch.float64, device=x.device)
    spare = torch.where(held, ids, x.shape[1])
    if s["log_sum"] is None:
        p = torch.softmax(torch.where(held, t, -math.inf), dim=1)
    else:
        p = torch.where(held, torch.exp(t - s["log_sum"][part].double()[:, None]), 0.0)
    target.scatter_(1, spare, p)
    target[:, -1] = 0.0
    log_q = torch.log_softmax(x / tau, dim=1)
    in_top = torch.zeros_like(target).scatter_(1, spare, 1.0)[:, :-1] > 0
    target = target[:, :-1]
    kl = (torch.xlogy(target, target) - target * torch.where(in_top, log_q, 0.0)).sum(dim=1)
    q = torch.exp(log_q)
    gradient = q * target.sum(dim=1, keepdim=True) - target
    if s["log_sum"] is not None:
        log_rest_q = torch.logsumexp(torch.where(in_top, -math.inf, log_q), dim=1)
        rest = torch.where(log_rest_q > -math.inf, (1.0 - target.sum(dim=1)).clamp(min=0.0), 0.0)
        kl = kl + torch.where(rest > 0, torch.xlogy(rest, rest) - rest * log_rest_q, 0.0)
        others = torch.where(in_top, 0.0, torch.exp(log_q - log_rest_q[:, None]))
        gradient = gradient + rest[:, None] * (q - others)
    loss = torch.where(weight == 0, 0.0, weight * tau * tau * kl)
    if not s["gradient"]:
        return loss
    return loss, torch.where(weight[:, None] == 0, 0.0, gradient * (weight * tau)[:, None])


_EXACT = {"adjust": _exact_adjust, "top": _exact_top, "distill": _exact_distill}
