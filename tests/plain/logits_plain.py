"""Rows of logits, token by token in 64 bits: penalties, biases and masks; a row's largest logits; a student's loss against a teacher's top
logits with its gradient. Loops over rows, Python numbers where it is no slower: nothing here is shared with the package."""

from __future__ import annotations

import math
from collections import Counter

import numpy as np


def adjust_row(x, prompt=(), answer=(), repetition=1.0, presence=0.0, frequency=0.0, biases=(), allowed=None):
    """`biases`: (token, value) pairs; `allowed`: a truth value per token, or None."""
    x = np.array(x, dtype=np.float64)
    counts = Counter(answer)
    for token in set(prompt) | set(answer):
        if 0 <= token < len(x):
            x[token] = x[token] / repetition if x[token] > 0 else x[token] * repetition
            if counts[token]:
                x[token] -= frequency * counts[token] + presence
    for token, value in biases:
        if 0 <= token < len(x):
            x[token] += value
    if allowed is not None:
        x[~np.asarray(allowed, dtype=bool)] = -math.inf
    return x


def top_row(x, k, temperature=1.0):
    x = np.array(x, dtype=np.float64)
    order = sorted(range(len(x)), key=lambda i: (0 if x[i] == x[i] else 1, -x[i] if x[i] == x[i] else 0.0, i))[:k]
    m = float(np.max(x))
    if math.isnan(m) or math.isinf(m):
        return x[order], order, m
    return x[order], order, m / temperature + math.log(np.exp((x - m) / temperature).sum())


def distill_row(x, ids, teacher, log_sum=None, temperature=1.0, weight=1.0):
    """(loss, gradient) of one row; entries outside the table are none."""
    x, v = np.array(x, dtype=np.float64), len(x)
    gradient = np.zeros(v)
    if weight == 0:
        return 0.0, gradient
    z = x / temperature
    with np.errstate(all="ignore"):
        z = z - z.max()
        log_q = z - math.log(np.exp(z).sum())
    q = np.exp(log_q)
    entries = [(int(i), float(t) / temperature) for i, t in zip(ids, teacher) if 0 <= i < v]
    if log_sum is None:
        finite = [t for _, t in entries if t > -math.inf]
        lse = max(finite) + math.log(sum(math.exp(t - max(finite)) for t in finite)) if finite else 0.0
    else:
        lse = float(log_sum)
    p = [(i, math.exp(t - lse) if t > -math.inf else 0.0, t - lse) for i, t in entries]
    mass = sum(pk for _, pk, _ in p)
    loss = sum(pk * (log_pk - log_q[i]) for i, pk, log_pk in p if pk > 0)
    for i, pk, _ in p:
        gradient[i] -= pk
    whole = mass
    if log_sum is not None:
        listed = np.zeros(v, dtype=bool)
        listed[[i for i, _, _ in p]] = True
        rest, rest_p = q[~listed].sum(), max(0.0, 1.0 - mass)
        if rest > 0 and rest_p > 0:
            loss += rest_p * (math.log(rest_p) - math.log(rest))
            gradient[~listed] -= rest_p * q[~listed] / rest
            whole += rest_p
    gradient += whole * q
    return weight * temperature**2 * loss, weight * temperature * gradient
