"""Workloads of the vocabulary-row operators of on-policy distillation.

Two operators on rows of logits: ``kl_div_topk`` (train or score a student on a teacher's listed
columns) and ``sample_tokens`` (temperature, top-k, top-p and min-p from given random numbers).
With ``own`` false, ``run`` computes them from elementary torch operations; with ``own`` true it
calls the framework's entry points.
"""

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"


def _d(name, n, v, k, dt="bf16", kind="logits", tail="renorm", reduction="mean", temp=1.0, train=True,
       ignored=0.0, idx64=False, scale=1.0):
    return {"name": name, "op": "distill", "n": n, "v": v, "k": k, "dt": dt, "kind": kind, "tail": tail,
            "reduction": reduction, "temp": temp, "train": train, "ignored": ignored, "idx64": idx64,
            "scale": scale}


def _s(name, n, v, dt="bf16", temp=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, banned=0, flat=False):
    return {"name": name, "op": "sample", "n": n, "v": v, "dt": dt, "temp": temp, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "mixed": mixed, "banned": banned, "flat": flat}


def listed():
    return [
        # the smallest training step: one packed micro-sequence of a small model, latency counts
        _d("distill_n16_v32000", 16, 32000, 64),
        # a micro-batch over a 32 K vocabulary, teacher's lists with their own log-sum-exp
        _d("distill_n8192_v32000", 8192, 32000, 64, tail="bucket", temp=2.0, ignored=0.05),
        # the large vocabulary: lists of 64 stored as probabilities next to 64-bit columns
        _d("distill_n4096_v128256", 4096, 128256, 64, kind="probs", tail="bucket", temp=2.0, idx64=True),
        # a vocabulary that is no multiple of a vector, fp16 with a loss scale, masked prompt rows
        _d("distill_n1021_v50257_fp16", 1021, 50257, 33, dt="fp16", ignored=0.2, scale=65536.0),
        # fp32 logits and long lists
        _d("distill_n1024_v128256_fp32", 1024, 128256, 256, dt="fp32", tail="drop"),
        # scoring a held-out batch: per-row values, no gradient
        _d("distill_score_n4096_v128256", 4096, 128256, 64, tail="bucket", reduction="none", train=False),
        # one sequence being answered, the usual nucleus
        _s("sample_n1_v128256_topp", 1, 128256, temp=0.8, top_p=0.95),
        # a small batch with the usual top-k in front of the nucleus
        _s("sample_n64_v32000_topk_topp", 64, 32000, temp=0.7, top_k=50, top_p=0.9),
        # a full serving batch, nucleus over the large vocabulary, some columns banned
        _s("sample_n256_v128256_topp", 256, 128256, temp=1.0, top_p=0.9, banned=200),
        # roll-outs of on-policy training: the plain distribution, odd vocabulary, fp32 logits
        _s("sample_n512_v50257_fp32", 512, 50257, dt="fp32"),
        # roll-outs that only cut the tail, near-uniform rows among the requests
        _s("sample_n512_v128256_minp", 512, 128256, min_p=0.02, flat=True),
        # a batch of requests that each bring their own settings, greedy ones among them
        _s("sample_n1024_v32000_mixed", 1024, 32000, mixed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _vocab(rng):
    if rng.random() < 0.4:
        return rng.choice([32000, 32001, 50257, 50304, 128256])
    return _log_int(rng, 1000, 160000)


def draw(rng):
    v = _vocab(rng)
    dt = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.5:
        n = _log_int(rng, 1, max(1, min(16384, 4096 * 128256 // (2 * v))))
        k = _log_int(rng, 1, 256)
        c = _d("", n, v, k, dt=dt, kind=rng.choice(["logits", "probs"]), tail=rng.choice(["renorm", "drop", "bucket"]),
               reduction=rng.choice(["mean", "sum", "none"]), temp=rng.choice([1.0, 1.0, 1.5, 2.0]),
               train=rng.random() < 0.75, ignored=rng.choice([0.0, 0.0, 0.1, 0.5]), idx64=rng.random() < 0.5,
               scale=65536.0 if dt == "fp16" else 1.0)
    else:
        n = _log_int(rng, 1, max(1, min(2048, 512 * 128256 // v)))
        filt = rng.choice(["none", "k", "p", "kp", "m", "all", "mixed"])
        c = _s("", n, v, dt=dt, temp=rng.choice([0.6, 0.8, 1.0, 1.0, 1.3]),
               top_k=_log_int(rng, 2, 500) if filt in ("k", "kp", "all") else 0,
               top_p=rng.uniform(0.5, 0.99) if filt in ("p", "kp", "all") else 1.0,
               min_p=rng.uniform(0.001, 0.2) if filt in ("m", "all") else 0.0,
               mixed=filt == "mixed", banned=rng.choice([0, 0, 50]), flat=rng.random() < 0.2)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _distill_inputs(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    n, v, k, dt = case["n"], case["v"], case["k"], _DT[case["dt"]]
    student = torch.empty(n, v, device=_DEV, dtype=dt)
    idx = torch.empty(n, k, device=_DEV, dtype=torch.int64)
    top = torch.empty(n, k, device=_DEV, dtype=torch.float32)
    lse = torch.empty(n, device=_DEV, dtype=torch.float32)
    step = max(1, (1 << 26) // v)
    for lo in range(0, n, step):
        s = 3 * torch.randn(min(step, n - lo), v, device=_DEV, generator=g)
        t = s + 0.5 * torch.randn(s.shape, device=_DEV, generator=g)
        student[lo:lo + step] = s.to(dt)
        top[lo:lo + step], idx[lo:lo + step] = torch.topk(t, k, dim=-1)
        lse[lo:lo + step] = torch.logsumexp(t / case["temp"], dim=-1)
    teacher = top
    if case["kind"] == "probs":
        teacher = torch.exp(top / case["temp"] - lse[:, None])
    elif dt != torch.float32:
        teacher = top.to(dt)               # logits are stored in the model's type
    if case["ignored"] > 0:                # prompt tokens and padding have no list
        gone = torch.rand(n, device=_DEV, generator=g) < case["ignored"]
        idx[gone] = -1
    up = torch.randn(n, device=_DEV, generator=g) if case["reduction"] == "none" else None
    need_lse = case["kind"] == "logits" and case["tail"] != "renorm"
    return {"student": student, "idx": idx if case["idx64"] else idx.to(torch.int32), "teacher": teacher,
            "lse": lse if need_lse else None, "up": up}


def _sample_inputs(case, seed):
    # a language model's next-token rows: a power law over a scrambled order of the vocabulary, of a
    # steepness of its own for each row, with noise on top
    g = torch.Generator(device=_DEV).manual_seed(seed)
    n, v, dt = case["n"], case["v"], _DT[case["dt"]]
    stride = next(s for s in range(v * 5 // 8 | 1, v * 5 // 8 + 1000) if math.gcd(s, v) == 1)
    steep = 1.0 + torch.rand(n, 1, device=_DEV, generator=g)
    if case["flat"]:
        steep[torch.rand(n, 1, device=_DEV, generator=g) < 0.25] = 0.05
    start = torch.randint(0, v, (n, 1), device=_DEV, generator=g)
    place = torch.arange(v, device=_DEV)[None, :] * stride
    logits = torch.empty(n, v, device=_DEV, dtype=dt)
    step = max(1, (1 << 26) // v)
    for lo in range(0, n, step):
        hi = min(n, lo + step)
        rank = (place + start[lo:hi]) % v
        x = 14.0 - steep[lo:hi] * torch.log1p(rank.float()) + 0.5 * torch.randn(hi - lo, v, device=_DEV, generator=g)
        logits[lo:hi] = x.to(dt)
    if case["banned"]:
        logits[:, torch.randint(0, v, (case["banned"],), device=_DEV, generator=g)] = -math.inf
    u = torch.rand(n, device=_DEV, generator=g)
    par = {key: case[key] for key in ("temp", "top_k", "top_p", "min_p")}
    if case["mixed"]:
        kind = torch.randint(0, 6, (n,), device=_DEV, generator=g)
        r = torch.rand(n, device=_DEV, generator=g)
        par["temp"] = torch.where(kind == 0, torch.zeros_like(r), 0.5 + r)
        par["top_k"] = torch.where((kind == 1) | (kind == 4), 1 + (r * 99).int(), torch.zeros_like(kind).int())
        par["top_p"] = torch.where((kind == 2) | (kind == 4), 0.5 + 0.49 * r, torch.ones_like(r))
        par["min_p"] = torch.where(kind == 3, 0.1 * r, torch.zeros_like(r))
    return {"logits": logits, "u": u, **par}


def prepare(case, seed):
    if case["op"] == "distill":
        state = _distill_inputs(case, seed)
        state["student"].requires_grad_(case["train"])
    else:
        state = _sample_inputs(case, seed)
    state["case"] = case
    return state


# ------------------------------------------------------------------ plain forms
def _plain_distill(st):
    c = st["case"]
    student, inv = st["student"].detach(), 1.0 / c["temp"]
    z = student.float() * inv
    idx = st["idx"].long()
    here = idx >= 0
    rows = here[:, 0]
    col = idx.clamp(min=0)
    # the divergence is a small difference of long sums: sums and the listed columns in 64 bits
    t = st["teacher"].double()
    if c["kind"] == "probs":
        q = torch.where(here, t, 0.0)
        if c["tail"] == "renorm":
            q = q / q.sum(-1, keepdim=True).clamp(min=1e-38)
    else:
        t = torch.where(here, t * inv, -math.inf)
        if c["tail"] == "renorm":
            q = torch.where(here, torch.exp(t - t.max(-1, keepdim=True).values), 0.0)
            q = q / q.sum(-1, keepdim=True).clamp(min=1e-38)
        else:
            q = torch.exp(t - st["lse"][:, None])
    m = z.max(-1, keepdim=True).values
    lse = m.double() + torch.log(torch.exp(z - m).sum(-1, keepdim=True, dtype=torch.float64))
    logp = student.gather(1, col).double() * inv - lse
    loss = torch.where(q > 0, q * (torch.log(q) - logp), 0.0).sum(-1)
    total = q.sum(-1, keepdim=True)
    rest = None
    if c["tail"] == "bucket":
        rest = (1.0 - total).clamp(min=0)
        listed_ = torch.zeros(z.shape, dtype=torch.bool, device=z.device).scatter_(1, col, here)
        zr = z.masked_fill(listed_, -math.inf)
        mr = zr.max(-1, keepdim=True).values
        lse_rest = mr.double() + torch.log(torch.exp(zr - mr).sum(-1, keepdim=True, dtype=torch.float64))
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - lse_rest + lse), 0.0)[:, 0]
        total = total + rest
    loss = torch.where(rows, loss, 0.0)
    n_valid = rows.sum().clamp(min=1).float()
    if c["reduction"] == "none":
        out, up = loss, st["up"][:, None]
    elif c["reduction"] == "sum":
        out, up = loss.sum(), 1.0
    else:
        out, up = loss.sum() / n_valid, 1.0 / n_valid
    if not c["train"]:
        return [out.float()]
    grad = torch.exp(z - lse.float()) * total.float()
    if rest is not None:
        grad = grad - rest.float() * torch.exp(zr - lse_rest.float())
    grad.scatter_add_(1, col, -q.float())
    grad = torch.where(rows[:, None], grad * (up * inv * c["scale"]), 0.0)
    return [out.float(), grad.to(student.dtype)]


def _as_column(x, like, dtype):
    # settings are held in 32 bits, whether they come as numbers or as tensors
    x = x if torch.is_tensor(x) else torch.full((like.shape[0],), x, device=like.device,
                                                dtype=torch.int32 if dtype == torch.int64 else torch.float32)
    return x.to(dtype)[:, None]


def _plain_sample(st):
    x = st["logits"]
    v = x.shape[1]
    temp = _as_column(st["temp"], x, torch.float64)
    top_k = _as_column(st["top_k"], x, torch.int64)
    top_p = _as_column(st["top_p"], x, torch.float64)
    min_p = _as_column(st["min_p"], x, torch.float64)
    # 64 bits: the running sums decide between neighbouring tokens
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    sorted_x = order.values.double()
    greedy = temp == 0
    e = torch.exp((sorted_x - sorted_x[:, :1]) / torch.where(greedy, 1.0, temp))
    rank = torch.arange(v, device=x.device)[None, :]
    keep = (top_k <= 0) | (rank < top_k)
    w = torch.where(keep, e, 0.0)
    run = torch.cumsum(w, -1)
    keep &= ((run - w) < top_p * run[:, -1:]) | (top_p >= 1)
    keep &= (e >= min_p) | (min_p <= 0)
    keep &= ~greedy | (rank == 0)
    w = torch.where(keep, e, 0.0)
    mass = torch.zeros_like(w).scatter_(1, order.indices, w)
    run = torch.cumsum(mass, -1)
    total = run[:, -1:]
    token = (run <= st["u"].double()[:, None] * total).sum(-1, keepdim=True)
    last = torch.where(mass > 0, rank, 0).max(-1, keepdim=True).values
    token = torch.minimum(token, last)
    logprob = torch.log(mass.gather(1, token) / total)[:, 0]
    return [token[:, 0], logprob.float()]


# ------------------------------------------------------------------ the framework's calls
def _own_distill(st):
    import forgeminds_amd as fm

    c, student = st["case"], st["student"]
    loss = fm.kernels.kl_div_topk(student, st["idx"], st["teacher"], teacher_lse=st["lse"],
                                  probs=c["kind"] == "probs", tail=c["tail"], reduction=c["reduction"],
                                  temperature=c["temp"])
    if not c["train"]:
        return [loss]
    up = st["up"] if c["reduction"] == "none" else torch.ones((), device=student.device)
    if c["scale"] != 1.0:
        up = up * c["scale"]
    (grad,) = torch.autograd.grad(loss, student, up)
    return [loss.detach(), grad]


def _own_sample(st):
    import forgeminds_amd as fm

    token, logprob = fm.kernels.sample_tokens(st["logits"], st["u"], temperature=st["temp"], top_k=st["top_k"],
                                              top_p=st["top_p"], min_p=st["min_p"])
    return [token, logprob]


def run(state):
    if state["case"]["op"] == "distill":
        return _own_distill(state) if own else _plain_distill(state)
    return _own_sample(state) if own else _plain_sample(state)


def work(case):
    n, v = case["n"], case["v"]
    size = 4 if case["dt"] == "fp32" else 2
    if case["op"] == "distill":
        lists = n * case["k"] * ((8 if case["idx64"] else 4) + (4 if case["kind"] == "probs" else size))
        moved = n * v * size * (2 if case["train"] else 1) + lists + 4
        return {"bytes": moved, "flops": n * v * (8 if case["train"] else 4)}
    # an exponential where the whole mass counts; with top-k alone a comparison
    return {"bytes": n * v * size + n * (4 + 8 + 4), "flops": n * v * (2 if case["top_k"] else 4)}


# ------------------------------------------------------------------ 64-bit values
def _exact_distill(case, seed):
    st = _distill_inputs(case, seed)
    n, T = case["n"], case["temp"]
    idx, teacher = st["idx"].long(), st["teacher"].double()
    valid = int((idx[:, 0] >= 0).sum().item())
    per_row = case["reduction"] == "none"
    grads, losses = [], []
    step = max(1, (1 << 26) // case["v"])
    for lo in range(0, n, step):
        z = st["student"][lo:lo + step].double() / T
        i, t = idx[lo:lo + step], teacher[lo:lo + step]
        used = i >= 0
        logp = torch.log_softmax(z, -1)
        if case["kind"] == "probs":
            q = t * used
        elif case["tail"] == "renorm":
            q = torch.softmax((t / T).masked_fill(~used, -1e300), -1) * used
        else:
            q = torch.exp(t / T - st["lse"][lo:lo + step].double()[:, None]) * used
        if case["tail"] == "renorm":
            q = q / q.sum(-1, keepdim=True).clamp(min=1e-300)
        # the teacher's distribution laid out over the vocabulary
        dense = torch.zeros_like(z)
        where = torch.zeros_like(z)
        dense.scatter_add_(1, i.clamp(min=0), q)
        where.scatter_add_(1, i.clamp(min=0), used.double())
        loss = (torch.xlogy(dense, dense) - dense * logp).sum(-1)
        grad = torch.exp(logp) * dense.sum(-1, keepdim=True) - dense
        if case["tail"] == "bucket":
            left = (1 - q.sum(-1, keepdim=True)).clamp(min=0)
            out = logp.masked_fill(where > 0, -math.inf)
            log_left = torch.logsumexp(out, -1, keepdim=True)
            loss = loss + (torch.xlogy(left, left) - left * log_left)[:, 0]
            grad = grad + torch.exp(logp) * left - torch.exp(out - log_left) * left
        live = used[:, 0]
        losses.append(torch.where(live, loss, 0.0))
        if case["train"]:
            up = st["up"][lo:lo + step].double()[:, None] if per_row else (
                1.0 / max(valid, 1) if case["reduction"] == "mean" else 1.0)
            grads.append(torch.where(live[:, None], grad / T * up * case["scale"], 0.0))
    loss = torch.cat(losses)
    if not per_row:
        loss = loss.sum() / (max(valid, 1) if case["reduction"] == "mean" else 1)
    return [loss, torch.cat(grads)] if case["train"] else [loss]


def _exact_sample(case, seed):
    st = _sample_inputs(case, seed)
    n = case["n"]
    x = st["logits"].double().cpu().numpy()

    def setting(key):
        val = st[key]
        return val.double().cpu().numpy() if torch.is_tensor(val) else np.full(n, np.float32(val), np.float64)
    temp, top_k, top_p, min_p = (setting(key) for key in ("temp", "top_k", "top_p", "min_p"))
    u = st["u"].double().cpu().numpy()
    token, logprob = np.zeros(n, np.int64), np.zeros(n)
    for i in range(n):
        row = x[i]
        best = int(np.argmax(row))
        if temp[i] == 0:
            token[i] = best
            continue
        e = np.exp((row - row[best]) / temp[i])
        kept = np.arange(row.size)
        if 0 < top_k[i] < row.size or top_p[i] < 1:
            kept = np.argsort(-row, kind="stable")
            if 0 < top_k[i] < row.size:
                kept = kept[:int(top_k[i])]
            if top_p[i] < 1:
                c = np.cumsum(e[kept])
                kept = kept[:1 + int(np.searchsorted(c[:-1], top_p[i] * c[-1], side="left"))]
        if min_p[i] > 0:
            kept = kept[e[kept] >= min_p[i]]
        kept = np.sort(kept)
        c = np.cumsum(e[kept])
        token[i] = kept[min(int(np.searchsorted(c, u[i] * c[-1], side="right")), kept.size - 1)]
        logprob[i] = math.log(e[token[i]] / c[-1])
    return [torch.from_numpy(token).to(_DEV), torch.from_numpy(logprob).to(_DEV)]


def exact(case, seed):
    return _exact_distill(case, seed) if case["op"] == "distill" else _exact_sample(case, seed)
