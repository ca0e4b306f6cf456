"""A beam search's selection on the CPU, request by request, with Python's own floats and sorting. Written apart
from the kernels; used by the tests alone."""
from __future__ import annotations

import math


def log_sum(x):
    """log sum exp x as a float, NaN where it has no value (a NaN, an infinity, or nothing above -infinity)."""
    if any(math.isnan(v) for v in x):
        return math.nan
    top = max(x)
    if math.isinf(top):
        return math.nan
    return top + math.log(math.fsum(math.exp(v - top) for v in x))


def select(logits, scores, done, end):
    """One request: logits [beams][vocab], scores, done [beams]; (score, beam, token, ended) of the best, in order.
    Within a beam the order is that of its logits, then of the tokens."""
    found = []
    for w, (x, s) in enumerate(zip(logits, scores)):
        if done[w]:
            found.append((-math.inf if math.isnan(s) else s, w, 0, end, True))
            continue
        total = log_sum(x)
        tokens = list(range(len(x)))
        if math.isnan(total) or math.isinf(s) or math.isnan(s):
            keys = [-math.inf] * len(x)
        else:
            tokens.sort(key=lambda v: (-x[v], v))
            keys = [s + (x[v] - total) for v in tokens]
        found += [(k, w, n, v, v == end) for n, (k, v) in enumerate(zip(keys, tokens))]
    found.sort(key=lambda c: (-c[0], c[1], c[2]))
    return [(k, w, v, e) for k, w, _, v, e in found[:len(scores)]]
