"""KL from a teacher's listed columns: ``kl_div_topk``, ``kl_distill_topk_loss`` and their entry points.

Tolerances, from the arithmetic of the sweep (u = 2^-24, half a step of fp32):
* a term exp2(x c - m) is off by a u ln2 for an argument of size a, and 2 u for the hardware exp2; a
  term of size 2^-a weighs 2^-a, so 16 u covers the row's sum; a thread adds up to P terms, each
  addition and each rescaling of the running sum within u: the log-sum-exp is within (P + 64) u
  (P = elements a thread sweeps, at most v / 256 for wide rows; the merge across threads is in 64 bits);
* the loss is sum q (log q - log p): within (P + 64) u of the truth for each of log p and log p_rest,
  plus 32 u for the rounding of log2(e) / T (relative to logits up to 32) and u |loss| for the store;
* a gradient element is a difference of terms whose sizes the oracle returns: each within
  (P + 64 + a) u, a <= 96 for the logits used here, plus half a step of the stored type.
"""

import ctypes
import math
import os
import re

import pytest
import torch

import forgeminds_amd as fm
from forgeminds_amd.kernels import _fallback as fb
from forgeminds_amd.kernels import _hip
from oracle import tokens as O

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def steps(v):
    return max(64, v // 256) + 64


def loss_tol(v, ref):
    return 2 * (steps(v) + 32) * U + 2 * U * ref.abs()


def make(n, v, k, dt=F32, kind="logits", tail="renorm", T=1.0, seed=0, idt=torch.int64, tdt=None, skipped=0, holes=0):
    g = torch.Generator().manual_seed(seed)
    s = 3 * torch.randn(n, v, generator=g)
    t = s + 0.5 * torch.randn(n, v, generator=g)
    s = s.to(dt)
    k_ = min(k, v)
    top, idx = torch.topk(t, k_, dim=-1)
    lse = torch.logsumexp(t / T, dim=-1)
    if k_ < k:      # more slots than columns: the rest is empty
        top = torch.cat([top, torch.zeros(n, k - k_)], -1)
        idx = torch.cat([idx, torch.full((n, k - k_), -1)], -1)
    for _ in range(holes):
        if k > 1:
            idx[torch.arange(n), torch.randint(1, k, (n,), generator=g)] = -1
    if skipped:
        idx[torch.arange(0, n, skipped)] = -1
    if kind == "probs":
        top = torch.exp(top / T - lse[:, None])
    top = top.to(tdt or F32)
    need = kind == "logits" and tail != "renorm"
    return s, idx.to(idt), top, (lse if need else None)


def call(s, idx, t, lse, kind, tail, T, reduction="mean", dev=None, **kw):
    mv = (lambda x: None if x is None else x.to(dev)) if dev else (lambda x: x)
    return fm.kernels.kl_div_topk(mv(s) if dev and s.device.type == "cpu" else s, mv(idx), mv(t), teacher_lse=mv(lse),
                                  probs=kind == "probs", tail=tail, reduction=reduction, temperature=T, **kw)


def check_grad(got, ref, size, dt, v, scale=1.0, what=""):
    got, ref, size = got.detach().double().cpu(), ref * scale, size * abs(scale)
    half = torch.finfo(dt).eps / 2
    quantum = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}[dt]
    bound = (steps(v) + 96) * U * size + half * ref.abs() * (1 + 1e-3) + quantum + 1e-38
    over = (got - ref).abs() - bound
    assert not torch.isnan(got).any(), what
    assert (over <= 0).all(), f"{what}: {int((over > 0).sum())} elements, worst by {over.max().item():.3g}"


# ------------------------------------------------------------------ oracle and host
@pytest.mark.parametrize("tail", ["renorm", "drop", "bucket"])
@pytest.mark.parametrize("kind", ["logits", "probs"])
def test_oracle_gradient_is_that_of_differences(kind, tail):
    s, idx, t, lse = make(3, 11, 4, torch.float64, kind, tail, 1.5, seed=1)
    s = s.double()
    args = dict(lse=lse, probs=kind == "probs", tail=tail, temperature=1.5)
    loss, grad, _size, _valid = O.kl_topk(s, idx, t, **args)
    h = 1e-5
    for j in range(11):
        d = torch.zeros_like(s)
        d[:, j] = h
        up, dn = O.kl_topk(s + d, idx, t, **args)[0], O.kl_topk(s - d, idx, t, **args)[0]
        assert torch.allclose((up - dn) / (2 * h), grad[:, j], atol=1e-8)


def test_whole_row_listed_is_the_full_kl():
    s, idx, t, _ = make(4, 9, 9, seed=2)
    full = torch.empty(4, 9).scatter_(1, idx, t)
    want = fm.kernels.kl_div_logits(s.double(), full.double(), "none", temperature=1.3)
    lse = torch.logsumexp(full / 1.3, -1)
    for tail in ("renorm", "drop", "bucket"):
        got = fm.kernels.kl_div_topk(s.double(), idx, t, teacher_lse=lse, tail=tail, reduction="none", temperature=1.3)
        assert torch.allclose(got, want, atol=1e-6), tail
    top_p = torch.exp(t / 1.3 - lse[:, None])
    got = fm.kernels.kl_div_topk(s.double(), idx, top_p, probs=True, tail="bucket", reduction="none", temperature=1.3)
    assert torch.allclose(got, want, atol=1e-6)


HOST = [(5, 7, 3, F32, "logits", "renorm", 1.0), (4, 100, 16, F32, "logits", "bucket", 2.0), (3, 33, 5, F32, "probs", "drop", 1.5),
        (6, 1, 1, F32, "logits", "renorm", 1.0), (3, 5, 9, F32, "probs", "bucket", 1.0), (4, 50, 8, BF16, "probs", "renorm", 0.7),
        (5, 64, 64, F32, "logits", "bucket", 1.0)]


@pytest.mark.parametrize("n,v,k,dt,kind,tail,T", HOST)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_torch_path_matches_the_oracle(n, v, k, dt, kind, tail, T, reduction):
    s, idx, t, lse = make(n, v, k, dt, kind, tail, T, seed=n + v, skipped=3, holes=1, idt=torch.int32)
    loss, grad, size, valid = O.kl_topk(s, idx, t, lse, kind == "probs", tail, T)
    s = s.requires_grad_(True)
    got = call(s, idx, t, lse, kind, tail, T, reduction)
    assert got.dtype == F32
    nv = max(int(valid.sum()), 1)
    want = {"mean": loss.sum() / nv, "sum": loss.sum(), "none": loss}[reduction]
    assert ((got.detach().double() - want).abs() <= n * loss_tol(v, want)).all()
    up = torch.randn(n, generator=torch.Generator().manual_seed(5)) if reduction == "none" else torch.tensor(1.0)
    (g,) = torch.autograd.grad(got, s, up)
    scale = up.double()[:, None] if reduction == "none" else torch.tensor([[1.0 / nv if reduction == "mean" else 1.0]]).double()
    check_grad(g, grad * scale, size * scale.abs(), dt, v)


def test_repeated_empty_and_outside_columns_on_the_torch_path():
    s = torch.randn(4, 6, dtype=torch.float64, generator=torch.Generator().manual_seed(3)).requires_grad_(True)
    idx = torch.tensor([[2, 2, 5, 2], [-1, 0, 1, 2], [0, -1, -7, 3], [1, 6, 2, 3]])
    q = torch.tensor([[.1, .2, .3, .15], [.5, .5, 0, 0], [.2, 9., 9., .6], [.1, .2, .3, .4]])
    for tail in ("renorm", "drop", "bucket"):
        got = fm.kernels.kl_div_topk(s, idx, q, probs=True, tail=tail, reduction="none")
        loss, grad, _s, _v = O.kl_topk(s, idx, q, probs=True, tail=tail)
        assert torch.allclose(got, loss, atol=1e-12, equal_nan=True) and got[3].isnan() and got[1] == 0
        (g,) = torch.autograd.grad(got[:3].sum(), s)
        assert torch.allclose(g[:3], grad[:3], atol=1e-12)


def test_refusals():
    s, idx, t, lse = make(3, 10, 4)
    bad = [dict(tail="rest"), dict(reduction="avg"), dict(temperature=0.0), dict(temperature=float("inf")),
           dict(temperature=float("nan")), dict(tail="drop"), dict(tail="bucket"),
           dict(tail="drop", teacher_lse=torch.zeros(2))]
    for kw in bad:
        with pytest.raises(ValueError):
            fm.kernels.kl_div_topk(s, idx, t, **kw)
    for a in [(s, idx.float(), t), (s, idx[:2], t[:2]), (s, idx, t[:, :3]), (s, idx[:, :0], t[:, :0]), (s, idx, t.long()),
              (s[:, :0], idx, t), (s.long(), idx, t), (s[0], idx, t), (s, idx.to("meta"), t)]:
        with pytest.raises(ValueError):
            fm.kernels.kl_div_topk(*a)
    with pytest.raises(ValueError):
        fm.kernels.kl_distill_topk_loss(torch.zeros(4, 2), torch.zeros(10, 2), idx, t)
    with pytest.raises(ValueError):
        fm.kernels.kl_distill_topk_loss(torch.zeros(3, 2), torch.zeros(10, 2), idx, t, chunk=0)


def test_no_rows_and_all_rows_skipped():
    s = torch.zeros(0, 8, requires_grad=True)
    e = fm.kernels.kl_div_topk(s, torch.zeros(0, 2, dtype=torch.int64), torch.zeros(0, 2))
    assert e.item() == 0
    s = torch.randn(2, 8).requires_grad_(True)
    loss = fm.kernels.kl_div_topk(s, torch.full((2, 3), -1), torch.randn(2, 3))
    loss.backward()
    assert loss.item() == 0 and (s.grad == 0).all()


def test_chunked_head_is_transparent_on_the_torch_path():
    g = torch.Generator().manual_seed(9)
    _s, idx, t, lse = make(10, 20, 5, tail="bucket", seed=4, skipped=4)
    outs = []
    for chunk in (3, 100):
        h = torch.randn(10, 6, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
        w = torch.randn(20, 6, generator=torch.Generator().manual_seed(2)).requires_grad_(True)
        loss = fm.kernels.kl_distill_topk_loss(h.view(2, 5, 6), w, idx.view(2, 5, 5), t.view(2, 5, 5),
                                               teacher_lse=lse.view(2, 5), tail="bucket", chunk=chunk)
        loss.backward()
        outs.append((loss.detach(), h.grad, w.grad))
    for a, b in zip(*outs):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    want = fm.kernels.kl_div_topk(h.detach() @ w.detach().t(), idx, t, teacher_lse=lse, tail="bucket")
    assert torch.allclose(outs[0][0], want, rtol=1e-5)
    assert fm.kernels.kl_distill_topk_loss(torch.zeros(0, 6), w, idx[:0], t[:0]).item() == 0


def test_declarations_exports_and_argument_validation():
    text = open(os.path.join(ROOT, "include", "fm_hip_tokens.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    decl = {m.group(1): m.group(2).count(",") + 1
            for m in re.finditer(r"\b(?:int|size_t)\s+(fm_[a-z_0-9]+)\s*\(([^;]*?)\)\s*;", text, flags=re.S)}
    assert set(decl) == set(_hip.TOKEN_SIGNATURES)
    if not os.path.exists(_hip.LIB_PATH):
        from forgeminds_amd import build
        build.build(verbose=False)
        _hip.reset_for_tests()
    lib = _hip.lib()
    for name, nargs in decl.items():
        assert len(_hip.TOKEN_SIGNATURES[name][1]) == nargs and hasattr(lib, name), name

    def fwd(n=4, v=8, k=2, dt=2, bits=64, tdt=0, kind=0, tail=0, T=1.0, red=2):
        return lib.fm_kl_topk_fwd(*(None,) * 8, n, v, k, dt, bits, tdt, kind, tail, T, red, None)

    def both(n=4, v=8, k=2, dt=2, bits=64, tdt=0, kind=0, tail=0, T=1.0, red=2):
        return lib.fm_kl_topk_loss_grad(*(None,) * 9, n, v, k, dt, bits, tdt, kind, tail, T, red, None)

    def bwd(n=4, v=8, k=2, dt=2, bits=64, tdt=0, kind=0, tail=0, T=1.0):
        return lib.fm_kl_topk_bwd(*(None,) * 7, 0, None, n, v, k, dt, bits, tdt, kind, tail, T, None)
    for f in (fwd, both, bwd):
        for kw in (dict(), dict(n=-1), dict(v=0), dict(k=0), dict(dt=5), dict(bits=16), dict(tdt=9), dict(kind=2),
                   dict(tail=3), dict(T=0.0), dict(T=float("nan")), dict(T=float("inf"))):
            assert f(**kw) == 1, (f.__name__, kw)
            assert lib.fm_last_error()
        assert f(k=1025) == 2 and f(v=2 ** 31) == 2
        assert f(n=2 ** 22) == 2 and f(v=2 ** 30) == 2
    assert both(red=0) == 1 and fwd(red=7) == 1 and bwd(n=0) == 0 and fwd(n=0, red=0) == 0
    # the gradient of saved stats needs a buffer of its own, and a gradient per row needs grad_out
    p = ctypes.c_void_p(64)
    assert lib.fm_kl_topk_bwd(p, p, p, None, p, None, None, 0, p, 4, 8, 2, 2, 64, 0, 1, 0, 1.0, None) == 1
    q = ctypes.c_void_p(128)
    assert lib.fm_kl_topk_bwd(p, p, p, None, p, None, None, 1, q, 4, 8, 2, 2, 64, 0, 1, 0, 1.0, None) == 1
    # teacher logits without their log-sum-exp
    assert lib.fm_kl_topk_bwd(p, p, p, None, p, None, None, 0, q, 4, 8, 2, 2, 64, 0, 0, 1, 1.0, None) == 1


# ------------------------------------------------------------------ GPU
GPU = [  # n, v, k, dtype, kind, tail, T, idx dtype, teacher dtype
    (5, 1, 1, F32, "logits", "renorm", 1.0, torch.int64, F32),
    (1, 1, 1, F32, "probs", "bucket", 1.0, torch.int64, F32),
    (7, 5, 9, F32, "logits", "bucket", 1.0, torch.int32, F32),
    (3, 64, 64, BF16, "probs", "bucket", 1.0, torch.int64, F32),
    (6, 1000, 7, F32, "logits", "drop", 1.5, torch.int64, F32),
    (300, 1003, 33, BF16, "logits", "renorm", 1.0, torch.int32, BF16),
    (9, 4099, 128, F16, "probs", "renorm", 2.0, torch.int64, F32),
    (9, 4099, 129, BF16, "logits", "bucket", 1.0, torch.int64, F16),
    (4, 8200, 1024, F32, "logits", "bucket", 2.0, torch.int32, F32),
    (6, 16392, 64, BF16, "probs", "drop", 1.0, torch.int32, F32),
    (40, 32000, 64, BF16, "logits", "bucket", 2.0, torch.int32, BF16),
    (8, 32001, 64, BF16, "probs", "bucket", 1.0, torch.int64, F32),
    (5, 50257, 33, F16, "logits", "renorm", 1.0, torch.int64, F16),
    (4, 50257, 300, F32, "probs", "bucket", 1.5, torch.int64, F32),
    (6, 65544, 64, BF16, "logits", "renorm", 1.0, torch.int64, F32),
    (6, 128256, 64, BF16, "probs", "bucket", 2.0, torch.int64, F32),
    (3, 128256, 256, F32, "logits", "drop", 1.0, torch.int64, F32),
    (2, 151937, 1000, F16, "probs", "bucket", 1.0, torch.int32, F32),
    (3, 200003, 64, BF16, "logits", "bucket", 1.0, torch.int64, F32),
    (2, 262147, 16, F32, "logits", "renorm", 1.0, torch.int64, F32),
]
gpu = pytest.mark.gpu


def to_dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@gpu
@pytest.mark.parametrize("n,v,k,dt,kind,tail,T,idt,tdt", GPU)
def test_loss_and_gradient_on_gpu(n, v, k, dt, kind, tail, T, idt, tdt):
    s, idx, t, lse = make(n, v, k, dt, kind, tail, T, seed=n + v + k, idt=idt, tdt=tdt, skipped=4 if n > 2 else 0,
                          holes=1 if k > 3 else 0)
    loss, grad, size, valid = O.kl_topk(s, idx, t, lse, kind == "probs", tail, T)
    nv = max(int(valid.sum()), 1)
    sd, di, dt_, dl = to_dev(s, idx, t, lse)
    fm.kernels.reset_stats()
    up = torch.randn(n, generator=torch.Generator().manual_seed(5))
    for reduction in ("mean", "sum", "none"):
        x = sd.clone().requires_grad_(True)
        got = call(x, di, dt_, dl, kind, tail, T, reduction)
        want = {"mean": loss.sum() / nv, "sum": loss.sum(), "none": loss}[reduction]
        tol = loss_tol(v, loss)
        tol = {"mean": tol.sum() / nv + 2 * U * want.abs(), "sum": tol.sum() + 2 * U * want.abs(), "none": tol}[reduction]
        assert ((got.detach().double().cpu() - want).abs() <= tol).all(), reduction
        s_ = {"mean": 1.0 / nv, "sum": 1.0}.get(reduction)
        g_in = up.to(DEV) if reduction == "none" else torch.ones((), device=DEV)
        scale = up.double()[:, None] if reduction == "none" else torch.full((1, 1), s_, dtype=torch.float64)
        if dt == F16:
            g_in, scale = g_in * 1024, scale * 1024
        (g,) = torch.autograd.grad(got, x, g_in)
        assert g.dtype == dt and g.shape == x.shape
        check_grad(g, grad * scale, size * scale.abs(), dt, v, what=reduction)
        assert torch.equal(x.detach(), sd)
        # scoring alone gives the same loss
        with torch.no_grad():
            only = call(x, di, dt_, dl, kind, tail, T, reduction)
        assert ((only.double().cpu() - want).abs() <= tol).all()
    assert fm.kernels.stats()["fallback"] == 0


@gpu
def test_gradient_written_in_place_retained_and_scaled():
    s, idx, t, lse = make(7, 9000, 20, BF16, "logits", "bucket", seed=3, skipped=3)
    loss, grad, size, valid = O.kl_topk(s, idx, t, lse, False, "bucket")
    nv = int(valid.sum())
    sd, di, td, dl = to_dev(s, idx, t, lse)
    x = sd.clone().requires_grad_(True)
    h = x * 1.0
    out = call(h, di, td, dl, "logits", "bucket", 1.0, reuse=True)
    (3.0 * out).backward()
    # the in-forward gradient is rounded once before and once after the factor of 3
    ref = grad * (3.0 / nv)
    assert ((x.grad.double().cpu() - ref).abs() <= 2.1 * 2 ** -8 * ref.abs() + (steps(9000) + 96) * U * size * 3 / nv + 1e-38).all()
    x2 = sd.clone().requires_grad_(True)
    out = call(x2, di, td, dl, "logits", "bucket", 1.0)
    out.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="already consumed"):
        out.backward()
    x3 = sd.clone().requires_grad_(True)
    out = call(x3, di, td, dl, "logits", "bucket", 1.0, retain=True)
    (a,) = torch.autograd.grad(out, x3, retain_graph=True)
    a = a.clone()
    (b,) = torch.autograd.grad(out, x3, retain_graph=True)
    assert torch.equal(a, b) and torch.equal(a, x2.grad)
    check_grad(a, grad, size, BF16, 9000, 1.0 / nv)


@gpu
@pytest.mark.parametrize("dt,v", [(F32, 300), (BF16, 20000), (BF16, 131080)])
def test_repeated_columns_and_columns_past_the_row(dt, v):
    n, k = 6, 200
    g = torch.Generator().manual_seed(1)
    s = torch.randn(n, v, generator=g).to(dt)
    idx = torch.randint(0, v, (n, k), generator=g)
    idx[0] = 7                                   # one column, k times
    idx[1, ::2] = idx[1, 1::2]                   # every column twice
    idx[2, 50:] = 0                              # padding by column 0 with probability 0
    idx[3] = torch.arange(k) // 3                # neighbours, three times each
    idx[4, 9] = v                                # past the row
    idx[5] = v - 1 - torch.arange(k)
    q = torch.rand(n, k, generator=g) / k
    q[2, 50:] = 0
    for tail in ("renorm", "drop", "bucket"):
        loss, grad, size, _ = O.kl_topk(s, idx, q, probs=True, tail=tail)
        x = s.to(DEV).requires_grad_(True)
        got = fm.kernels.kl_div_topk(x, idx.to(DEV), q.to(DEV), probs=True, tail=tail, reduction="none")
        ok = [0, 1, 2, 3, 5]
        assert got[4].isnan()
        assert ((got.detach().double().cpu() - loss).abs() <= loss_tol(v, loss))[ok].all()
        (gr,) = torch.autograd.grad(got, x, torch.ones(n, device=DEV), retain_graph=True)
        check_grad(gr[ok], grad[ok], size[ok], dt, v, 1.0, tail)
        assert gr[4].isnan().all()
        (g2,) = torch.autograd.grad(got, x, torch.ones(n, device=DEV))
        assert torch.equal(gr[ok], g2[ok])       # the order inside the table changes nothing
        y = s.to(DEV).requires_grad_(True)
        one = fm.kernels.kl_div_topk(y[:4], idx[:4].to(DEV), q[:4].to(DEV), probs=True, tail=tail, reduction="sum")
        one.backward()
        check_grad(y.grad[:4], grad[:4], size[:4], dt, v, 1.0, tail)


@gpu
def test_masked_logits_far_tails_and_whole_rows():
    v = 5000
    g = torch.Generator().manual_seed(2)
    s = torch.randn(5, v, generator=g)
    s[0, 100:] = -float("inf")                   # most of the vocabulary masked
    s[1, 30:] = -300.0                           # the unlisted columns far below the listed ones
    s[2, 64:] = torch.finfo(F32).min             # masked with the type's lowest value
    s[3] = s[3] * 20
    idx = torch.arange(64)[None, :].repeat(5, 1)
    idx[1, 30:] = -1
    q = torch.softmax(torch.randn(5, 64, generator=g), -1)
    q[2] = q[2] / q[2].double().sum()
    q[[0, 1, 3, 4]] *= 0.9
    rows = [0, 1, 3, 4]
    loss, grad, size, _ = O.kl_topk(s[rows], idx[rows], q[rows], probs=True, tail="bucket")
    x = s.to(DEV).requires_grad_(True)
    got = fm.kernels.kl_div_topk(x, idx.to(DEV), q.to(DEV), probs=True, tail="bucket", reduction="none")
    # logits of size 300: the rounding of log2(e)/T is relative to them
    assert ((got.detach().double().cpu()[rows] - loss).abs() <= loss_tol(v, loss) + 2 * 512 * U).all()
    (gr,) = torch.autograd.grad(got[rows].sum(), x)
    a, b = gr[rows].double().cpu(), grad
    assert ((a - b).abs() <= (steps(v) + 96 + 512) * U * size + U * b.abs() + 1e-37).all()
    assert (gr[0, 100:] == 0).all()
    loss, grad, size, _ = O.kl_topk(s[[0, 2]], idx[[0, 2]], q[[0, 2]], probs=True, tail="renorm")
    y = s[[0, 2]].to(DEV).requires_grad_(True)
    got = fm.kernels.kl_div_topk(y, idx[[0, 2]].to(DEV), q[[0, 2]].to(DEV), probs=True, tail="renorm", reduction="sum")
    got.backward()
    assert abs(got.item() - loss.sum().item()) <= loss_tol(v, loss).sum().item()
    check_grad(y.grad, grad, size, F32, v)


@gpu
def test_nan_logits_stay_in_their_row():
    s, idx, t, _ = make(3, 700, 5, F32, seed=8)
    s[1, 400] = float("nan")
    x = s.to(DEV).requires_grad_(True)
    got = fm.kernels.kl_div_topk(x, idx.to(DEV), t.to(DEV), reduction="none")
    (g,) = torch.autograd.grad(got, x, torch.ones(3, device=DEV))
    assert got[1].isnan() and not got[[0, 2]].isnan().any()
    assert g[1].isnan().all() and not g[[0, 2]].isnan().any()


@gpu
def test_unaligned_strided_and_batched_inputs():
    s, idx, t, lse = make(12, 1001, 9, BF16, "logits", "bucket", seed=6, skipped=5)
    loss, grad, size, valid = O.kl_topk(s, idx, t, lse, False, "bucket")
    nv = int(valid.sum())
    sd, di, td, dl = to_dev(s, idx, t, lse)
    flat = torch.zeros(12 * 1001 + 3, device=DEV, dtype=BF16)
    off = flat[3:].view(12, 1001)                 # a base that is not 16-byte aligned
    off.copy_(sd)
    wide = torch.zeros(12, 1100, device=DEV, dtype=BF16)
    wide[:, 50:1051] = sd
    for x in (off, wide[:, 50:1051], sd.view(3, 4, 1001), sd.view(4, 3, 1001).transpose(0, 1).contiguous().transpose(0, 1)):
        lead = x.shape[:-1]
        leaf = x.detach().requires_grad_(True)
        got = call(leaf, di.view(*lead, 9), td.view(*lead, 9), dl.view(lead), "logits", "bucket", 1.0)
        assert abs(got.item() - loss.sum().item() / nv) <= loss_tol(1001, loss).sum().item() / nv + 1e-9
        (g,) = torch.autograd.grad(got, leaf)
        check_grad(g.reshape(12, 1001), grad, size, BF16, 1001, 1.0 / nv)
        rows = call(leaf, di.view(*lead, 9), td.view(*lead, 9), dl.view(lead), "logits", "bucket", 1.0, "none")
        assert rows.shape == lead


@gpu
def test_runs_are_bit_identical_on_any_stream_and_replay_in_a_graph():
    s, idx, t, lse = make(300, 32000, 64, BF16, "logits", "bucket", 2.0, seed=7, skipped=9)
    sd, di, td, dl = to_dev(s, idx, t, lse)
    want = _hip.kl_topk_loss_grad(sd, di, td, dl, False, "bucket", 2.0, "mean")
    want = [w.clone() for w in want]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _hip.kl_topk_loss_grad(sd, di, td, dl, False, "bucket", 2.0, "mean")
        _hip.kl_topk_fwd(sd, di, td, dl, False, "bucket", 2.0, "mean")
    torch.cuda.synchronize()
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    xs = sd.clone()
    with torch.cuda.graph(graph):
        loss, grad, _rows = _hip.kl_topk_loss_grad(xs, di, td, dl, False, "bucket", 2.0, "mean")
        sl, _r, stats, nv = _hip.kl_topk_fwd(xs, di, td, dl, False, "bucket", 2.0, "mean")
        back = _hip.kl_topk_bwd(xs, di, td, dl, stats, nv, None, False, False, "bucket", 2.0)
    for turn in range(3):
        xs.copy_(sd if turn != 1 else sd.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        e_loss, e_grad, _ = _hip.kl_topk_loss_grad(xs, di, td, dl, False, "bucket", 2.0, "mean")
        e_sl, _r2, e_stats, e_nv = _hip.kl_topk_fwd(xs, di, td, dl, False, "bucket", 2.0, "mean")
        e_back = _hip.kl_topk_bwd(xs, di, td, dl, e_stats, e_nv, None, False, False, "bucket", 2.0)
        assert torch.equal(loss, e_loss) and torch.equal(grad, e_grad) and torch.equal(sl, e_sl)
        assert torch.equal(back, e_back)


@gpu
def test_produced_lists_train_a_head():
    # the teacher's lists as the framework produces them, stored, then trained on through a head
    g = torch.Generator().manual_seed(11)
    n, d, v, k, T = 70, 64, 4000, 32, 2.0
    h = torch.randn(n, d, generator=g)
    w = 0.3 * torch.randn(v, d, generator=g)
    teacher = 2 * torch.randn(n, v, generator=g)
    hd, wd, td = h.to(DEV), w.to(DEV), teacher.to(DEV)
    student = hd @ wd.t()
    _l, probs, idx = fm.kernels.kl_div_logits_topk(student, td, k, temperature=T, index_dtype=torch.int32)
    idx[::6] = -1
    ha, wa = hd.clone().requires_grad_(True), wd.clone().requires_grad_(True)
    loss = fm.kernels.kl_distill_topk_loss(ha, wa, idx, probs, probs=True, tail="bucket", temperature=T, chunk=32)
    loss.backward()
    hb, wb = h.double().requires_grad_(True), w.double().requires_grad_(True)
    ref = fb.kl_div_topk(hb @ wb.t(), idx.cpu(), probs.cpu(), None, True, "bucket", "mean", T)
    ref.backward()
    # fp32 products of 64 terms of size one and of n rows: 64 u and n u on gradients of this size
    assert abs(loss.item() - ref.item()) <= 1e-4 * abs(ref.item())
    for a, b in ((ha.grad, hb.grad), (wa.grad, wb.grad)):
        assert ((a.double().cpu() - b).abs() <= 1e-4 * b.abs().max()).all()


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_small_bucket_losses_keep_their_digits(dt):
    """The unlisted columns hold nearly all mass, listed ones have twice the student's probability: a
    loss of 1e-4 that is a difference of terms of size 1. With d_r, d_l the relative errors of the two
    running sums the loss is off by (p_r - q_r) d_r + p_l d_l, and |p_r - q_r| = p_l. At 2048 columns a
    thread adds 8 weights or 16: arguments below 16 in base 2 are rounded by 2^-21 (3.3e-7 of the
    weight), the exponential by 2^-23, a rescale by 2^-23, at most 16 adds by 2^-24 each: 1.6e-6. The
    scale's own rounding, 2^-24, shifts sum (q - p) z by less than 2 * 16 * 2^-24 * p_l. Together below
    2 * 1.6e-6 * p_l + 2e-6 * p_l, and the fp32 result's 2^-24.
    """
    n, v, k, T = 64, 2048, 4, 2.0
    g = torch.Generator().manual_seed(5)
    s = (torch.randn(n, v, generator=g) * 1.5).to(dt)
    p = torch.softmax(s.double() / T, 1)
    pl, idx = p.topk(k, dim=1, largest=False)
    q = (2 * pl).float()
    ref = O.kl_topk(s, idx, q, None, True, "bucket", T)[0]
    got = fm.kernels.kl_div_topk(*to_dev(s, idx, q), probs=True, tail="bucket", temperature=T, reduction="none")
    tol = 5.2e-6 * pl.sum(1) + ref.abs() * 2.0 ** -23
    err = (got.double().cpu() - ref).abs()
    assert (err <= tol).all(), (err / tol).max()


@gpu
def test_rows_past_two_to_the_31_elements():
    # rows repeat every 64: the same loss and gradient wherever they stand
    n, v, k, m = 16800, 128256, 32, 64
    assert n * v > 2 ** 31
    g = torch.Generator().manual_seed(8)
    s = (2 * torch.randn(m, v, generator=g)).to(BF16)
    t, idx = (s.float() + 0.5 * torch.randn(m, v, generator=g)).topk(k)
    lse = torch.logsumexp(t, 1) + 0.3
    rows = torch.arange(n, device=DEV) % m
    sd, idx, t, lse = to_dev(s, idx, t, lse)
    big = sd.repeat((n + m - 1) // m, 1)[:n].requires_grad_(True)
    for reduction in ("none", "sum"):
        big.grad = None
        loss = fm.kernels.kl_div_topk(big, idx[rows], t[rows], teacher_lse=lse[rows], tail="bucket", reduction=reduction)
        loss.sum().backward()
        small = sd.clone().requires_grad_(True)
        want = fm.kernels.kl_div_topk(small, idx, t, teacher_lse=lse, tail="bucket", reduction="none")
        want.sum().backward()
        if reduction == "none":
            assert (loss - want[rows]).abs().max() <= 2.0 ** -20 * want.abs().max()
        for at in (0, 37, 2 ** 31 // v - 1, 2 ** 31 // v, 2 ** 31 // v + 1, n - 1):
            a, b = big.grad[at].float(), small.grad[at % m].float()
            assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-30).all(), (reduction, at)


@gpu
def test_another_device_than_the_current_one_is_refused_or_served():
    s, idx, t, _ = make(2, 50, 3)
    with pytest.raises(ValueError):
        fm.kernels.kl_div_topk(s.to(DEV), idx, t.to(DEV))
    with pytest.raises(ValueError):
        fm.kernels.kl_div_topk(s.to(DEV), idx.to(DEV), t)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("v", [1000, 4096, 8200, 16384])
def test_the_mean_counts_every_row(dt, v):
    """The gradient of the mean is divided by the rows that have a list, however many rows there are
    beside the threads of a workgroup and whichever of them are skipped."""
    n, k = 257, 64
    s, idx, t, lse = make(n, v, k, dt, "logits", "renorm", seed=v)
    _loss, grad, size, _valid = O.kl_topk(s, idx, t)
    sd, di, td = to_dev(s, idx, t)
    for m in (1, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257):
        for skipped in (range(0), range(0, m, 3), range(min(m, 64)), range(min(m, 128)), range(64, m), range(1, m)):
            live = torch.ones(m, dtype=torch.bool)
            live[list(skipped)] = False
            gone = torch.where(live.to(DEV)[:, None], di[:m], -1)
            x = sd[:m].clone().requires_grad_(True)
            fm.kernels.kl_div_topk(x, gone, td[:m]).backward()
            scale = live[:, None].double() / max(int(live.sum()), 1)
            check_grad(x.grad, grad[:m] * scale, size[:m] * scale, dt, v, what=f"{m} rows, {m - int(live.sum())} skipped")


def agrees(got, want, tol):
    """Within ``tol``, or both past the largest fp32 value."""
    got = got.detach().double().cpu()
    return (((got - want).abs() <= tol) | ((got == float("inf")) & torch.isinf(want.float()))).all()


def low_reference(s, idx, q, T):
    """Row losses and gradient of their sum for tail="bucket", float64, from differences to the maxima
    (``oracle.tokens`` goes through log p, where 3e38 leaves no digit of the other terms)."""
    n, v = s.shape
    loss, grad, size = torch.zeros(n), torch.zeros(n, v), torch.zeros(n, v)
    loss, grad, size = loss.double(), grad.double(), size.double()
    for i in range(n):
        z, c, w = s[i].double() / T, idx[i], q[i].double()
        m = z.max()
        p = torch.exp(z - m)
        ls = torch.log(p.sum())
        p = p / p.sum()
        out = torch.ones(v, dtype=torch.bool)
        out[c] = False
        left = max(0.0, 1.0 - math.fsum(w.tolist()))
        mr = z[out].max()
        share = torch.where(out, torch.exp(z - mr), 0.0)
        ls_r = torch.log(share.sum())
        loss[i] = (w * (torch.log(w) - ((z[c] - m) - ls))).sum() + left * (math.log(left) - ((mr - m) + (ls_r - ls)))
        share = share / share.sum()
        grad[i] = p * (w.sum() + left) - left * share
        size[i] = p * (w.sum() + left) + left * share
        grad[i, c] -= w
        size[i, c] += w
    return loss, grad / T, size / T


@gpu
@pytest.mark.parametrize("T", [0.7, 1.0, 2.0])
@pytest.mark.parametrize("dt,v", [(F32, 300), (BF16, 300), (BF16, 5003), (F32, 70001), (BF16, 140000)])
def test_bucket_over_logits_masked_with_the_lowest_value(dt, v, T):
    """Finite rows have a finite gradient, however low their masks. Where the low logits take part the
    loss is q_r times 3.4e38 / T: off by the rounding of log2(e) / T and of the result, half a step each,
    and of q_r, which the reference shares. A loss past the largest fp32 value is rounded to inf (at
    T = 0.7 listed probabilities of 0.9 at masked logits: 4.4e38)."""
    k, low = 64, torch.finfo(dt).min
    g = torch.Generator().manual_seed(v)
    s = torch.randn(7, v, generator=g)
    idx = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(7)])
    q = torch.softmax(torch.randn(7, k, generator=g), -1) * 0.9
    out = torch.ones(7, v, dtype=torch.bool).scatter_(1, idx, False)
    s[0][out[0]] = low                                # everything unlisted masked
    s[1][out[1]] = low
    q[1] = q[1] * (1 - 2.0 ** -20) / q[1].double().sum()        # a bucket of rounding
    s[2] = low                                        # the whole row masked: even
    s[3][out[3]] = low                                # some of the unlisted ones out altogether
    s[3, ::2] = torch.where(out[3, ::2], -float("inf"), s[3, ::2])
    s[4][~out[4]] = low                               # everything listed masked
    s[5][~out[5]] = low                               # half as low outside
    s[5][out[5]] = low / 2
    s = s.to(dt)
    loss, grad, size = low_reference(s, idx, q, T)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()
    tol = loss_tol(v, loss) + U * loss.abs()
    sd, di, dq = to_dev(s, idx, q)
    odd = torch.zeros(7 * v + 1, device=DEV, dtype=dt)[1:].view(7, v)
    odd.copy_(sd)
    kw = dict(probs=True, tail="bucket", temperature=T)
    for base in (sd, odd):
        x = base.detach().requires_grad_(True)
        rows = fm.kernels.kl_div_topk(x, di, dq, reduction="none", **kw)
        assert agrees(rows, loss, tol)
        (gr,) = torch.autograd.grad(rows, x, torch.ones(7, device=DEV))
        check_grad(gr, grad, size, dt, v, what="from stats")
        total = fm.kernels.kl_div_topk(x, di, dq, reduction="sum", **kw)
        assert agrees(total, loss.sum(), tol.sum() + U * loss.sum().abs())
        (gr,) = torch.autograd.grad(total, x)
        check_grad(gr, grad, size, dt, v, what="with the loss")
    h = sd.clone().requires_grad_(True)
    (gr,) = torch.autograd.grad(fm.kernels.kl_div_topk(h * 1.0, di, dq, reduction="sum", reuse=True, **kw), h)
    check_grad(gr, grad, size, dt, v, what="in place")
    # the other tails: the whole row is one sum
    for tail in ("drop", "renorm"):
        x = sd[[2, 6]].clone().requires_grad_(True)
        rows = fm.kernels.kl_div_topk(x, di[[2, 6]], dq[[2, 6]], probs=True, tail=tail, reduction="none", temperature=T)
        ref = O.kl_topk(s[[2, 6]], idx[[2, 6]], q[[2, 6]], None, True, tail, T)
        assert ((rows.detach().double().cpu() - ref[0]).abs() <= loss_tol(v, ref[0])).all()
        (gr,) = torch.autograd.grad(rows, x, torch.ones(2, device=DEV))
        check_grad(gr, ref[1], ref[2], dt, v, what=tail)


@gpu
@pytest.mark.parametrize("level", [-1e4, -1e6, -1e8, -1e9, -3e9, -1e12, -1e30, 1e9, 3e38])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_rows_at_one_far_level(dt, level):
    # whatever the level of a row, or of its unlisted columns, or of its listed ones (the sum at 3e38 is 4.3e38)
    n, v, k, T = 4, 3001, 32, 1.0
    g = torch.Generator().manual_seed(6)
    s = torch.randn(n, v, generator=g)
    idx = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    q = torch.softmax(torch.randn(n, k, generator=g), -1) * 0.5
    out = torch.ones(n, v, dtype=torch.bool).scatter_(1, idx, False)
    s[0] = level
    s[1][out[1]] = level
    s[2][~out[2]] = level
    s[3] = torch.where(torch.rand(v, generator=g) < 0.5, level, -abs(level) * 1.1)
    s = s.to(dt)
    loss, grad, size = low_reference(s, idx, q, T)
    tol = loss_tol(v, loss) + U * loss.abs()
    sd, di, dq = to_dev(s, idx, q)
    x = sd.clone().requires_grad_(True)
    for reduction in ("none", "sum"):
        out = fm.kernels.kl_div_topk(x, di, dq, probs=True, tail="bucket", reduction=reduction)
        want, t = (loss, tol) if reduction == "none" else (loss.sum(), tol.sum() + U * loss.sum().abs())
        assert agrees(out, want, t)
        (gr,) = torch.autograd.grad(out.sum(), x)
        check_grad(gr, grad, size, dt, v, what=reduction)


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("dt,v", [(F32, 40), (BF16, 3000)])
def test_a_row_without_a_finite_logit_has_no_gradient_to_give(dt, v, dev):
    # -inf everywhere is no distribution: loss and gradient are NaN, listed or not, in that row alone
    s, idx, t, _ = make(3, v, 5, dt, seed=4)
    s[1] = -float("inf")
    for tail, kw in (("renorm", {}), ("bucket", {"teacher_lse": torch.full((3,), 9.0, device=dev)})):
        for reduction in ("none", "sum"):
            x = s.to(dev).requires_grad_(True)
            out = fm.kernels.kl_div_topk(x, idx.to(dev), t.to(dev), tail=tail, reduction=reduction, **kw)
            (g,) = torch.autograd.grad(out.sum(), x)
            assert out.isnan()[1].item() if reduction == "none" else out.isnan().item()
            assert g[1].isnan().all() and not g[[0, 2]].isnan().any(), (tail, reduction)


@gpu
@pytest.mark.parametrize("dt,v,k", [(F32, 300, 64), (BF16, 3000, 64), (BF16, 40000, 256), (F32, 9000, 1024), (BF16, 131080, 1000)])
def test_the_order_of_the_slots_changes_no_bit(dt, v, k):
    # neighbouring columns share vectors and threads; probabilities are multiples of 2^-24, so their sums
    # are exact in any order
    n = 6
    g = torch.Generator().manual_seed(v + k)
    s = 3 * torch.randn(n, v, generator=g)
    idx = torch.stack([torch.arange(k) * step % v for step in (1, 2, 3, 5, 7, 1)])
    idx[5] = v - 1 - torch.arange(k)
    q = torch.randint(1, 2 ** 24 // k - 1, (n, k), generator=g).float() * 2.0 ** -24
    live = torch.ones(n, k, dtype=torch.bool)
    for i in range(n):                       # repeated columns (a step that wraps): one of them stays
        seen = set()
        for j in range(k):
            c = int(idx[i, j])
            live[i, j] = c not in seen
            seen.add(c)
    idx = torch.where(live, idx, -1)
    sd, di, dq = to_dev(s.to(dt), idx, q)
    want = None
    for turn in range(4):
        order = torch.randperm(k, generator=g)
        order = torch.cat([torch.zeros(1, dtype=torch.int64), order[order != 0]]) if turn else torch.arange(k)
        o = order.to(DEV)
        runs = []
        for _ in range(2):
            x = sd.clone().requires_grad_(True)
            rows = fm.kernels.kl_div_topk(x, di[:, o], dq[:, o], probs=True, tail="bucket", reduction="none")
            (g1,) = torch.autograd.grad(rows, x, torch.ones(n, device=DEV))
            y = sd.clone().requires_grad_(True)
            total = fm.kernels.kl_div_topk(y, di[:, o], dq[:, o], probs=True, tail="bucket", reduction="sum")
            (g2,) = torch.autograd.grad(total, y)
            runs.append((rows.detach(), g1, total.detach(), g2))
        want = want or runs[0]
        for got in runs:
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


@gpu
def test_students_past_two_to_the_33_elements_run_on_the_kernel():
    # 17 GB of logits and as much gradient, rows that repeat every 64
    n, v, k, m = 67000, 128256, 16, 64
    assert n * v > 2 ** 33
    g = torch.Generator().manual_seed(9)
    s = (2 * torch.randn(m, v, generator=g)).to(BF16)
    t, idx = (s.float() + 0.5 * torch.randn(m, v, generator=g)).topk(k)
    idx[5::9] = -1
    rows = torch.arange(n, device=DEV) % m
    sd, idx, t = to_dev(s, idx, t)
    big = sd.repeat((n + m - 1) // m, 1)[:n].requires_grad_(True)
    live = (idx[rows, 0] >= 0).sum()
    fm.kernels.reset_stats()
    loss = fm.kernels.kl_div_topk(big, idx[rows], t[rows])
    (grad,) = torch.autograd.grad(loss, big, torch.tensor(2.0 ** 17, device=DEV))
    assert fm.kernels.stats()["fallback"] == 0
    small = sd.clone().requires_grad_(True)
    each = fm.kernels.kl_div_topk(small, idx, t, reduction="none")
    (want,) = torch.autograd.grad(each, small, (2.0 ** 17 / live).expand(m))
    total = each.detach().double()[rows].sum() / live
    assert abs(loss.item() - total.item()) <= 2.0 ** -22 * total.item()
    for at in (0, 5, 2 ** 31 // v, 2 ** 32 // v, 2 ** 33 // v - 1, 2 ** 33 // v, n - 1):
        a, b = grad[at].float(), want[at % m].float()
        assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-30).all() and (at % m == 5) == (not b.any()), at


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("tail", ["renorm", "drop", "bucket"])
def test_what_a_skipped_row_holds_does_not_matter(tail, dev):
    # slot 0 is empty: NaN, infinities and columns past the row in what else the row holds change nothing
    nan, inf = float("nan"), float("inf")
    g = torch.Generator().manual_seed(3)
    s = torch.randn(7, 12, generator=g)
    idx = torch.randint(0, 12, (7, 3), generator=g)
    idx[1:6, 0] = -1
    t = torch.rand(7, 3, generator=g) * 0.3
    lse = torch.full((7,), 4.0)
    s[1], s[2], s[3, 5] = nan, -inf, inf
    idx[4, 1] = 12
    t[5, 1], t[5, 2], lse[5] = nan, inf, -inf
    for probs in (False, True):
        for reduction in ("none", "sum", "mean"):
            x = s.to(dev).requires_grad_(True)
            out = fm.kernels.kl_div_topk(x, idx.to(dev), t.to(dev), teacher_lse=lse.to(dev), probs=probs, tail=tail,
                                         reduction=reduction)
            (got,) = torch.autograd.grad(out.sum(), x)
            assert torch.isfinite(out).all() and torch.isfinite(got).all() and (got[1:6] == 0).all(), (probs, reduction)
            assert (got[[0, 6]] != 0).any(dim=-1).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
def test_temperatures_past_fp32(dev):
    # any positive finite number: past 1e30 the student is even and the loss log v minus the list's entropy
    s, idx, _t, _ = make(4, 500, 6, seed=2)
    q = torch.softmax(torch.randn(4, 6, generator=torch.Generator().manual_seed(1)), -1)
    want = math.log(500) + (q.double() * torch.log(q.double())).sum(-1)
    for T in (1e32, 3.5e38, 1e200):
        x = s.to(dev).requires_grad_(True)
        rows = fm.kernels.kl_div_topk(x, idx.to(dev), q.to(dev), probs=True, tail="drop", reduction="none", temperature=T)
        assert ((rows.detach().double().cpu() - want).abs() <= loss_tol(500, want) + (1 - q.double().sum(-1)).abs() * 7).all()
        (g,) = torch.autograd.grad(rows.sum(), x)
        assert (g.abs() <= 1.1 / T).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_the_loss_may_be_added_to_in_place(reduction, dt, dev):
    s, idx, t, _ = make(6, 300, 4, dt, seed=3)
    grads = []
    for inplace in (False, True):
        x = s.to(dev).view(2, 3, 300).requires_grad_(True)
        loss = fm.kernels.kl_div_topk(x, idx.view(2, 3, 4).to(dev), t.view(2, 3, 4).to(dev), reduction=reduction)
        aux = (x.float() ** 2).sum()
        if inplace:
            loss += aux
            loss *= 3.0
        else:
            loss = (loss + aux) * 3.0
        grads.append(torch.autograd.grad(loss.sum(), x)[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("T", [0.7, 1.0, 2.0])
@pytest.mark.parametrize("dt", [F32, BF16, torch.float64])
def test_bucket_over_the_lowest_values_on_the_torch_path(dt, T):
    v, k, low = 300, 64, torch.finfo(BF16 if dt == BF16 else F32).min
    g = torch.Generator().manual_seed(v)
    s = torch.randn(7, v, generator=g)
    idx = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(7)])
    q = torch.softmax(torch.randn(7, k, generator=g), -1) * 0.9
    out = torch.ones(7, v, dtype=torch.bool).scatter_(1, idx, False)
    s[0][out[0]] = low
    s[1][out[1]] = low
    s[1, ::2] = torch.where(out[1, ::2], -float("inf"), s[1, ::2])
    s[2] = low
    s[4][~out[4]] = low
    s[5][~out[5]] = low
    s[5][out[5]] = low / 2
    s = s.to(dt)
    loss, grad, size = low_reference(s, idx, q, T)
    for reduction in ("none", "sum"):
        x = s.clone().requires_grad_(True)
        got = fm.kernels.kl_div_topk(x, idx, q, probs=True, tail="bucket", temperature=T, reduction=reduction)
        assert got.dtype == (torch.float64 if dt == torch.float64 else F32)
        tol = loss_tol(v, loss) + U * loss.abs()
        assert agrees(got, loss, tol) if reduction == "none" else agrees(got, loss.sum(), tol.sum() + U * loss.sum().abs())
        (gr,) = torch.autograd.grad(got.sum(), x)
        check_grad(gr, grad, size, F32 if dt == torch.float64 else dt, v, what=reduction)


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("T", [1e20, 2e38, 1e45, 1e200])
def test_masked_logits_at_far_temperatures(T, dev):
    # even over what the mask leaves: loss log 500 minus the list's entropy, -inf columns without gradient
    n, v = 3, 1000
    s = torch.randn(n, v, generator=torch.Generator().manual_seed(5))
    s[:, 1::2] = -float("inf")
    idx = torch.arange(0, 12, 2).repeat(n, 1)
    q = torch.softmax(torch.randn(n, 6, generator=torch.Generator().manual_seed(6)), -1)
    want = math.log(500) * q.double().sum(-1) + (q.double() * torch.log(q.double())).sum(-1)
    for reduction in ("none", "sum"):
        x = s.to(dev).requires_grad_(True)
        got = fm.kernels.kl_div_topk(x, idx.to(dev), q.to(dev), probs=True, tail="drop", temperature=T, reduction=reduction)
        ref = want if reduction == "none" else want.sum()
        assert ((got.detach().double().cpu() - ref).abs() <= 3 * loss_tol(v, ref)).all()
        (g,) = torch.autograd.grad(got.sum(), x)
        assert not g.isnan().any() and (g[:, 1::2] == 0).all()
