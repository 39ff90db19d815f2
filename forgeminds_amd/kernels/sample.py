"""``sample_tokens``: one token per row of logits, with temperature, top-k, top-p and min-p, from given
uniform numbers, in one HIP launch.

Nothing like it exists in the reference, whose kernel package stops at ``topk`` and ``softmax``
(``forgemind/kernels/topk.py:273-297``, ``softmax.py:118-139``); the order of equal logits is that of
its ``topk`` (``topk.py:13-16``). Random numbers are an input, so that a row's token depends on nothing
but the row, its settings and its number: not on the batch, the launch or the device's generator. (The
kernel sums weights as integers, multiples of 2^-46 of the largest for rows of up to 2^17 columns.)
"""

from __future__ import annotations

import math

import torch

from . import _fallback as fb
from . import _hip
from ._common import _note, fast_ok, tracing

#: widest row of the kernel path; wider ones run the torch expression
MAX_VOCAB = 1 << 20
#: rows of one launch; more are drawn by several
MAX_ROWS = (1 << 22) - 1


def _setting(name: str, x, lead, like: torch.Tensor, dtype):
    """A number as it is, a tensor as a dense ``[rows]`` one of ``dtype``."""
    if not torch.is_tensor(x):
        return x
    if x.shape != lead:
        raise ValueError(f"{name} must be a number or a tensor {tuple(lead)}, got {tuple(x.shape)}")
    if x.device != like.device:
        raise ValueError(f"{name} is on {x.device}, the logits on {like.device}")
    if x.is_floating_point() != dtype.is_floating_point or x.dtype == torch.bool or x.is_complex():
        raise ValueError(f"{name} must be {'floating point' if dtype.is_floating_point else 'an integer'}, got {x.dtype}")
    if dtype == torch.int32 and x.dtype.itemsize >= 4 and x.dtype != torch.int32:
        x = x.to(torch.int64).clamp(-1, 2 ** 31 - 1)
    return x.detach().to(dtype).contiguous().view(-1)


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``(token, logprob)`` for each row of ``logits [..., V]`` and each number of ``u [...]`` in ``[0, 1)``.

    ``temperature``, ``top_k``, ``top_p`` and ``min_p`` are numbers, or tensors ``[...]`` with a setting
    per row; they are held in 32 bits. In this order:

    * the logits are divided by ``temperature``; 0 takes the first maximum, whatever the filters;
    * ``top_k``: only the ``k`` largest stay, equal ones in the order of their index (0, or ``V`` and
      more: all stay);
    * ``top_p``: the most probable stay until their mass reaches ``top_p`` of what top-k left, at least
      one (1: all stay);
    * ``min_p``: only tokens at least ``min_p`` times as probable as the most probable stay (0: all).

    ``token`` (int64) is the first index, ascending, at which the running mass of what stays exceeds
    ``u`` times the whole; ``logprob`` (fp32) is the token's log-probability among what stays. Weights
    and sums are held in 64 bits, and a row gives the same bits whatever rows come with it. A row without a distribution (it holds a NaN or ``+inf`` or nothing but
    ``-inf``, or its temperature tensor holds a negative, infinite or NaN value) gets ``-1`` and NaN.
    Neither output is differentiable.

    Traced calls (``torch.compile``) and rows wider than ``MAX_VOCAB`` run the torch expression: a 64-bit
    sort of every row.
    """
    if logits.dim() < 1 or logits.shape[-1] == 0 or not logits.is_floating_point():
        raise ValueError(f"sample_tokens needs floating-point logits [..., V], got {tuple(logits.shape)} {logits.dtype}")
    lead = logits.shape[:-1]
    if u.shape != lead or not u.is_floating_point():
        raise ValueError(f"u must be floating point {tuple(lead)}, got {tuple(u.shape)} {u.dtype}")
    if u.device != logits.device:
        raise ValueError(f"u is on {u.device}, the logits on {logits.device}")
    if not torch.is_tensor(temperature) and not 0 <= temperature <= torch.finfo(torch.float32).max:
        raise ValueError(f"temperature must be finite in 32 bits and not negative, got {temperature}")
    if not torch.is_tensor(top_k) and (not 0 <= top_k < math.inf or int(top_k) != top_k):
        raise ValueError(f"top_k must be a non-negative integer, got {top_k}")
    for name, x in (("top_p", top_p), ("min_p", min_p)):
        if not torch.is_tensor(x) and not 0 <= x <= 1:
            raise ValueError(f"{name} must be between 0 and 1, got {x}")
    v = logits.shape[-1]
    if not torch.is_tensor(top_k):
        top_k = min(int(top_k), 2 ** 31 - 1)
    f32 = torch.float32
    settings = [_setting("temperature", temperature, lead, logits, f32), _setting("top_k", top_k, lead, logits, torch.int32),
                _setting("top_p", top_p, lead, logits, f32), _setting("min_p", min_p, lead, logits, f32)]
    x2 = logits.detach().reshape(-1, v) if logits.numel() else logits.detach().reshape(0, v)
    u1 = u.detach().to(f32).contiguous().view(-1)

    def torch_path():
        cols = [s if torch.is_tensor(s) else torch.full((x2.shape[0],), s, device=x2.device,
                                                        dtype=torch.int32 if i == 1 else f32)
                for i, s in enumerate(settings)]
        token, logprob = fb.sample_tokens(x2, u1, *(c.unsqueeze(-1) for c in cols))
        return token.view(lead), logprob.view(lead)

    if logits.numel() == 0 or v > MAX_VOCAB or tracing():
        _note("sample_tokens shape")
        return torch_path()
    if not fast_ok(logits):
        return torch_path()
    x2, n = x2.contiguous(), x2.shape[0]
    if n <= MAX_ROWS:
        token, logprob = _hip.sample(x2, u1, *settings)
    else:
        parts = [_hip.sample(x2[lo:lo + MAX_ROWS], u1[lo:lo + MAX_ROWS],
                             *(s[lo:lo + MAX_ROWS] if torch.is_tensor(s) else s for s in settings))
                 for lo in range(0, n, MAX_ROWS)]
        token, logprob = (torch.cat(t) for t in zip(*parts))
    return token.view(lead), logprob.view(lead)


__all__ = ["sample_tokens", "MAX_VOCAB", "MAX_ROWS"]
