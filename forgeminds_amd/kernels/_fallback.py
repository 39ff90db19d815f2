"""The torch expressions the kernels stand in for.

This is what runs for CPU tensors, for float64, and under ``set_backend("fallback")`` -- the
same contract as the reference's ``forgemind/kernels/_fallback.py``: accumulate in fp32 for
half-precision inputs (float64/float32 keep their own precision) and round once, at the
output cast.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F


def _wide(t: torch.Tensor) -> torch.Tensor:
    """fp32 for half types, unchanged for float32/float64 (reference ``_fallback.py:15-23``)."""
    return t.float() if t.dtype in (torch.float16, torch.bfloat16) else t


def rms_norm(x, w, eps: float = 1e-6):
    """Reference ``_fallback.py:26-30``."""
    xw = _wide(x)
    inv = torch.rsqrt(xw.square().mean(dim=-1, keepdim=True) + eps)
    return (xw * inv * _wide(w)).to(x.dtype)


def add_rms_norm(x, delta, w, eps: float = 1e-6):
    """Reference ``_fallback.py:33-35``: the sum is rounded to x's dtype before it is normalised."""
    summed = x + delta
    return summed, rms_norm(summed, w, eps)


def layer_norm(x, w, b=None, eps: float = 1e-5):
    """``F.layer_norm`` in the wide dtype, one rounding (the rule of ``rms_norm`` above)."""
    xw = _wide(x)
    out = torch.nn.functional.layer_norm(xw, (x.shape[-1],), _wide(w).to(xw.dtype),
                                         None if b is None else _wide(b).to(xw.dtype), eps)
    return out.to(x.dtype)


def add_layer_norm(x, delta, w, b=None, eps: float = 1e-5):
    """The sum is rounded to x's dtype before it is normalised."""
    summed = x + delta
    return summed, layer_norm(summed, w, b, eps)


def kl_div_logits(student, teacher, reduction: str = "mean", temperature: float = 1.0):
    """KL(teacher || student) over the last dim (reference ``_fallback.py:52-69``).

    Differentiable wrt ``student`` through ordinary autograd; the teacher is detached.
    ``temperature`` divides both logit tensors first (no T**2 factor).
    """
    s, t = _wide(student), _wide(teacher).detach()
    if temperature != 1.0:
        s, t = s / temperature, t / temperature
    log_s = torch.log_softmax(s, dim=-1)
    log_t = torch.log_softmax(t, dim=-1)
    rows = (log_t.exp() * (log_t - log_s)).sum(dim=-1)
    if reduction == "none":
        return rows
    if reduction == "sum":
        return rows.sum()
    return rows.sum() / max(rows.numel(), 1)


def kl_div_topk(student, idx, teacher, teacher_lse=None, probs: bool = False, tail: str = "renorm",
                reduction: str = "mean", temperature: float = 1.0):
    """KL(teacher || student) from the teacher's values at the listed columns ``idx [..., k]``.

    Rows whose first slot is negative are skipped, other negative slots are empty, a repeated
    column counts once with the sum of its probabilities, a column past the row gives NaN.
    """
    live = idx[..., 0] >= 0
    # a skipped row holds anything: nothing of it may meet a gradient of zero
    idx = torch.where(live.unsqueeze(-1), idx, -1)
    s = torch.where(live.unsqueeze(-1), _wide(student), 0.0)
    if not 1 <= temperature <= 1e38:       # the lowest fp32 value (a mask) divided by it leaves fp32, or it does itself
        s = s.double()
    z = s / temperature
    v = s.shape[-1]
    logp = torch.log_softmax(z, dim=-1)
    used = idx >= 0
    col = idx.long().clamp(0, v - 1)
    # the teacher's few values in the widest type at hand
    t = torch.where(used, teacher.detach().double(), 0.0)
    if not probs:
        if tail == "renorm":
            t = torch.where(used, t / temperature, -float("inf"))
            t = torch.exp(t - torch.where(used[..., :1], t.amax(dim=-1, keepdim=True), 0.0))
        else:
            t = torch.where(used, torch.exp(t / temperature - teacher_lse.detach().double().unsqueeze(-1)), 0.0)
    if tail == "renorm":
        t = torch.where(used[..., :1], t / t.sum(dim=-1, keepdim=True), 0.0)
    t = torch.where((idx >= v).any(dim=-1, keepdim=True), float("nan"), t)
    q = torch.zeros_like(logp).scatter_add(-1, col, t.to(logp.dtype))
    rows = torch.where(q == 0, 0.0, q * (torch.log(torch.where(q == 0, 1.0, q)) - logp)).sum(dim=-1)
    if tail == "bucket":
        listed = torch.zeros(logp.shape, dtype=torch.int32, device=logp.device).scatter_add(-1, col, used.int()) > 0
        left = (1.0 - t.sum(dim=-1)).clamp(min=0).to(logp.dtype)
        left = torch.where(listed.all(dim=-1) | (left == 0), 0.0, left)
        some = left != 0
        # rows without a bucket take a finite stand-in, so that no gradient meets an infinity
        out = torch.where(some.unsqueeze(-1), z.masked_fill(listed, -float("inf")), z)
        # sums against maxima of their own: next to a mask's 3e38 the log of a sum has no digit left
        top, top_out = (t.detach().amax(dim=-1, keepdim=True) for t in (z, out))
        top_out = torch.where(torch.isinf(top_out), 0.0, top_out)
        log_rest = ((top_out - top).squeeze(-1) + torch.logsumexp(out - top_out, dim=-1)
                    - torch.logsumexp(z - top, dim=-1))
        rows = rows + torch.where(some, left * (torch.log(torch.where(some, left, 1.0)) - log_rest), 0.0)
    rows = torch.where(live, rows, 0.0)
    dtype = torch.promote_types(student.dtype, torch.float32)
    if reduction == "none":
        return rows.to(dtype)
    total = rows.sum().to(dtype)
    if reduction == "mean":
        total = total / live.sum().clamp(min=1).to(total.dtype)
    return total


def cross_entropy(logits, labels, ignore_index: int = -100, reduction: str = "mean"):
    """fp32 loss of ``F.cross_entropy`` summed over valid rows (reference ``loss.py:63-70``).

    ``mean`` divides by ``max(1, #valid)``. The math runs in fp32 on the logits' values, so a
    bf16 input does not get a bf16-rounded loss.
    """
    total = F.cross_entropy(_wide(logits), labels, ignore_index=ignore_index, reduction="sum")
    total = total.float()
    if reduction == "sum":
        return total
    n_valid = (labels != ignore_index).sum().clamp(min=1).to(torch.float32)
    return total / n_valid


def swiglu(gate, up):
    """Reference ``_fallback.py:48-49``."""
    return (F.silu(_wide(gate)) * _wide(up)).to(gate.dtype)


def swiglu_split(gate_up):
    half = gate_up.shape[-1] // 2
    return swiglu(gate_up[..., :half], gate_up[..., half:])


def qk_norm_rope(x, w, cos, sin, eps: float = 1e-6):
    """Per-head RMSNorm then half-split RoPE, x ``[B, T, H, D]`` (reference ``_fallback.py:38-45``)."""
    xw = _wide(x)
    inv = torch.rsqrt(xw.square().mean(dim=-1, keepdim=True) + eps)
    y = xw * inv * _wide(w)
    a, b = y.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1).to(x.dtype)


def topk_canonical(x, k: int):
    """Top-k in the canonical order (value desc, index asc inside ties, NaN largest).

    ``torch.topk`` promises no tie order, so the torch path gets it from a stable sort.
    """
    key = torch.nan_to_num(_wide(x), nan=float("inf"), posinf=float("inf"))
    # NaN and +inf share the top key; NaN must still come first, so rank NaN above +inf
    bump = torch.isnan(x)
    order = torch.sort(torch.where(bump, torch.zeros_like(key), torch.ones_like(key)),
                       dim=-1, stable=True).indices           # NaN first, original order inside
    key_sorted = torch.gather(key, -1, order)
    nan_sorted = torch.gather(bump, -1, order)
    # stable descending sort by value keeps (NaN first, then ascending index) inside ties
    composite = torch.where(nan_sorted, torch.full_like(key_sorted, float("inf")), key_sorted)
    second = torch.sort(composite, dim=-1, descending=True, stable=True).indices
    idx = torch.gather(order, -1, second)[..., :k]
    return torch.gather(x, -1, idx), idx


def sample_tokens(x, u, temp, top_k, top_p, min_p):
    """Token and log-probability per row of ``x [n, v]``; the settings are ``[n, 1]`` tensors.

    64-bit weights and sums, like the kernel: a border between two tokens must not move.
    """
    n, v = x.shape
    if x.numel() == 0:
        return x.new_zeros(n, dtype=torch.int64), x.new_zeros(n, dtype=torch.float32)
    temp, top_p, min_p = temp.double(), top_p.double(), min_p.double().clamp(max=1.0)
    order = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    m = order.values[:, :1]
    fine = torch.isfinite(m) & ~torch.isnan(x).any(dim=-1, keepdim=True) & (temp >= 0) & (temp < float("inf"))
    greedy = temp == 0
    safe_m = torch.where(fine, m, 0.0)
    gap = torch.where(fine, order.values - safe_m, 0.0)
    e = torch.exp(gap / torch.where(greedy | ~fine, 1.0, temp))
    rank = torch.arange(v, device=x.device)[None, :]
    keep = (top_k <= 0) | (top_k >= v) | (rank < top_k)
    w = torch.where(keep, e, 0.0)
    run = torch.cumsum(w, -1)
    keep = keep & (~(top_p < 1) | (rank == 0) | ((run - w) < top_p * run[:, -1:]))
    keep = keep & (~(min_p > 0) | (e >= min_p))
    keep = torch.where(greedy, rank == 0, keep)
    mass = torch.zeros_like(w).scatter_(1, order.indices, torch.where(keep, e, 0.0))
    run = torch.cumsum(mass, -1)
    total = run[:, -1:]
    u = torch.where(u > 0, u, 0.0).clamp(max=1.0 - 2.0 ** -24).double().unsqueeze(-1)
    token = torch.minimum((run <= u * total).sum(-1, keepdim=True),
                          torch.where(mass > 0, rank, 0).max(-1, keepdim=True).values)
    logprob = torch.log(mass.gather(1, token) / total)
    return (torch.where(fine, token, -1).squeeze(-1),
            torch.where(fine, logprob, float("nan")).squeeze(-1).float())
