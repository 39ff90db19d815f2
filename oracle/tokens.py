"""CPU oracles of the token-level operators -- TEST INFRASTRUCTURE, NOT PRODUCT CODE.

Row by row in 64 bits, from the operators' definitions. The reference has neither operator: parity
unpinned. ``tests/test_kl_topk.py`` pins the distillation one against differences, against
``torch.autograd`` and against the full-row KL; ``tests/test_sample.py`` pins the sampler against
brute force.
"""

import math

import numpy as np
import torch


def teacher_list(idx, teacher, v, lse=None, probs=False, tail="renorm", temperature=1.0):
    """One row: {column: probability} of the used slots, or None for a skipped row, "bad" when a
    column lies past the row."""
    idx = [int(c) for c in idx]
    if idx[0] < 0:
        return None
    if any(c >= v for c in idx):
        return "bad"
    vals = [(c, float(t)) for c, t in zip(idx, teacher) if c >= 0]
    if probs:
        w = [t for _, t in vals]
    elif tail == "renorm":
        top = max(t for _, t in vals)
        w = [math.exp((t - top) / temperature) for _, t in vals]
    else:
        w = [math.exp(t / temperature - float(lse)) for _, t in vals]
    if tail == "renorm":
        s = math.fsum(w)
        w = [x / s for x in w]
    q = {}
    for (c, _), x in zip(vals, w):
        q[c] = q.get(c, 0.0) + x
    return q


def kl_topk(student, idx, teacher, lse=None, probs=False, tail="renorm", temperature=1.0):
    """Per-row loss [n], gradient [n, v] of the row losses' sum and the size of the terms the gradient
    is a difference of [n, v], float64; valid rows [n] bool."""
    n, v = student.shape
    loss, grad, size = np.zeros(n), np.zeros((n, v)), np.zeros((n, v))
    valid = np.zeros(n, bool)
    x = student.detach().double().cpu().numpy()
    for i in range(n):
        q = teacher_list(idx[i].tolist(), teacher[i].double().tolist(), v, None if lse is None else lse[i].item(),
                         probs, tail, temperature)
        if q is None:
            continue
        valid[i] = True
        if q == "bad":
            loss[i], grad[i] = np.nan, np.nan
            continue
        z = x[i] / temperature
        m = z.max()
        logp = z - m - math.log(np.exp(z - m).sum())
        p = np.exp(logp)
        cols = np.array(sorted(q))
        qs = np.array([q[c] for c in cols])
        out = np.ones(v, bool)
        out[cols] = False
        left = max(0.0, 1.0 - math.fsum(qs)) if tail == "bucket" and out.any() else 0.0
        total = math.fsum(qs) + left
        loss[i] = math.fsum(a * (math.log(a) - logp[c]) for c, a in zip(cols, qs) if a > 0)
        grad[i] = p * total
        size[i] = p * total
        grad[i, cols] -= qs
        size[i, cols] += qs
        if left > 0:
            mr = z[out].max()
            lp_rest = mr - m + math.log(np.exp(z[out] - mr).sum()) + (logp[0] - (z[0] - m))
            loss[i] += left * (math.log(left) - lp_rest)
            share = np.exp(logp[out] - lp_rest)
            grad[i, out] -= left * share
            size[i, out] += left * share
    return (torch.from_numpy(loss), torch.from_numpy(grad / temperature), torch.from_numpy(size / temperature),
            torch.from_numpy(valid))
