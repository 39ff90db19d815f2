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


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: (token, logprob, margin). ``margin`` is how far, relative to the mass, the nearest
    decision (the cut of top-p, the border of the token) is from falling otherwise."""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or not np.isfinite(x.max()) or not 0 <= temperature < math.inf:
        return -1, math.nan, 1.0
    if temperature == 0:
        return int(np.argmax(x)), 0.0, 1.0
    with np.errstate(over="ignore"):
        e = np.exp((x - x.max()) / temperature)
    order = sorted(range(x.size), key=lambda j: (-x[j], j)) if x.size < 5000 else list(np.argsort(-x, kind="stable"))
    margin = 1.0
    if 0 < top_k < x.size:
        order = order[:top_k]
    if top_p < 1:
        total = math.fsum(e[order])
        goal = top_p * total
        before, kept = 0.0, []
        run = np.concatenate([[0.0], np.cumsum(e[order])])
        kept = [j for r, j in enumerate(order) if r == 0 or run[r] < goal]
        if top_p > 0:
            margin = min(margin, float(np.abs(run[1:-1] - goal).min()) / total if len(order) > 1 else 1.0)
        order = kept
    if min_p > 0:
        order = [j for j in order if e[j] >= min(min_p, 1.0)]
    order = np.array(sorted(order))
    run = np.cumsum(e[order])
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    r = u * run[-1]
    at = int(np.searchsorted(run, r, side="right"))
    if u > 0 and order.size > 1:
        margin = min(margin, float(np.abs(run[:-1] - r).min()) / run[-1])
    at = min(at, int(np.nonzero(e[order])[0][-1]))
    return int(order[at]), math.log(e[order[at]] / run[-1]), margin
