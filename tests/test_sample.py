"""``sample_tokens`` and ``fm_sample`` against the 64-bit oracle, row by row.

Tokens have to be equal wherever the arithmetic decides. The kernel's weights are within 1.1e-12, the
masses top-p is cut by are sums of up to v weights rounded to 2^-45 (v up to 2^17; finer for smaller
ones), half a step of that each: v 2^-46 = 1.9e-9 of a mass of at least 1 in the worst case. A decision
(the cut of top-p, the border of the token) nearer than DELTA to falling otherwise may do so: there the
token has to be that of u and top_p moved by at most DELTA. The log-probability is a 64-bit value
rounded to fp32: half a step, 2^-24 relative, plus 1e-11, plus the mass such a cut may move.
"""

import ctypes

import numpy as np
import pytest
import torch

import forgeminds_amd as fm
from forgeminds_amd.kernels import _hip
from oracle import tokens as O

DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


def zipf(n, v, seed, dt=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    steep = 0.3 + 1.7 * torch.rand(n, 1, generator=g)
    rank = torch.stack([torch.randperm(v, generator=g) for _ in range(n)]).float()
    x = (14 - steep * torch.log1p(rank) + 0.5 * torch.randn(n, v, generator=g)) * scale
    return x.to(dt), torch.rand(n, generator=g)


DELTA = 2.5e-9


def either(x, u, temperature, top_k, top_p, min_p):
    """The (token, logprob) pairs that decisions within DELTA allow; one pair almost always."""
    want = O.sample(x, u, temperature, top_k, top_p, min_p)
    if want[2] >= DELTA:
        return [want[:2]]
    ps = (top_p,) if not 0 < top_p < 1 else (top_p - DELTA, top_p, top_p + DELTA)
    return [want[:2]] + [O.sample(x, u + d, temperature, top_k, q, min_p)[:2] for d in (-DELTA, 0, DELTA) for q in ps]


def check_row(x, u, token, logprob, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    settings = (float(np.float32(temperature)), int(top_k), float(np.float32(top_p)), float(np.float32(min_p)))
    allowed = either(np.asarray(x, np.float64), u, *settings)
    near = [lp for t, lp in allowed if t == token]
    assert near, (token, allowed)
    if token < 0:
        assert np.isnan(logprob)
    else:
        assert any(abs(logprob - lp) <= 2.0 ** -24 * abs(lp) + 1e-11 + (2 * DELTA if len(allowed) > 1 else 0) for lp in near)


def check(x, u, tok, lp, **settings):
    xs = x.detach().double().cpu().numpy()
    for i in range(x.shape[0]):
        check_row(xs[i], u[i].item(), tok[i].item(), lp[i].item(),
                  **{k: (s[i].item() if torch.is_tensor(s) else s) for k, s in settings.items()})


SETTINGS = [dict(), dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=50), dict(top_k=1000),
            dict(top_p=0.9), dict(top_p=0.0), dict(top_p=0.999999), dict(min_p=0.05), dict(min_p=1.0),
            dict(temperature=1.7, top_k=40, top_p=0.8), dict(top_k=300, top_p=0.95, min_p=0.01),
            dict(temperature=0.05, top_k=20), dict(temperature=30.0, top_p=0.5), dict(temperature=0.01, top_p=0.9)]


# ------------------------------------------------------------------ host
@pytest.mark.parametrize("kw", SETTINGS)
@pytest.mark.parametrize("v", [1, 2, 9, 1000])
def test_torch_path_matches_the_oracle(v, kw):
    x, u = zipf(6, v, v)
    tok, lp = fm.kernels.sample_tokens(x, u, **kw)
    assert tok.dtype == torch.int64 and lp.dtype == F32
    check(x, u, tok, lp, **kw)


def test_oracle_against_brute_force():
    # the empirical distribution over an even grid of u is the filtered distribution
    x = torch.tensor([0.3, 2.0, -1.0, 2.0, 1.2, -float("inf")])
    p = torch.softmax(x.double() / 0.8, -1).numpy()
    order = [1, 3, 4, 0, 2, 5]
    cases = [(dict(), range(6)), (dict(top_k=2), [1, 3]), (dict(top_k=1), [1]),
             (dict(top_p=float(p[1]) * 1.5), [1, 3]), (dict(top_p=float(p[1]) * 0.5), [1]),
             (dict(min_p=float(p[4] / p[1]) * 0.99), [1, 3, 4]), (dict(top_k=4, top_p=0.999), order[:4])]
    for kw, kept in cases:
        q = np.zeros(6)
        q[list(kept)] = p[list(kept)]
        q /= q.sum()
        n = 4000
        hits = np.zeros(6)
        for j in range(n):
            t, lp, _m = O.sample(x.numpy(), (j + 0.5) / n, 0.8, **kw)
            hits[t] += 1
            assert abs(lp - np.log(q[t])) < 1e-9
        assert np.abs(hits / n - q).max() <= 1.0 / n, kw


def special_rows(v=300):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(F32).min
    g = torch.Generator().manual_seed(5)
    x = torch.randn(12, v, generator=g)
    x[0] = -inf                       # nothing left by the mask
    x[1, 7] = nan
    x[2, 9] = inf
    x[3] = low                        # masked with the type's lowest value: still a distribution
    x[4, :-1] = -inf                  # one column left
    x[5, 3:] = -inf
    x[6] = 1.5                        # all equal
    x[7] = torch.randint(0, 3, (v,), generator=g).float()      # few values
    x[8, ::2] = low
    x[9, 0], x[9, 1] = 0.0, -0.0
    x[9, 2:] = -1.0
    x[10] *= 1e30
    x[11, 5] = 1e4                    # an outlier far above the rest
    u = torch.tensor([.5, .5, .5, .37, .2, .7, .613, .41, .83, .5, .3, .9])
    return x, u


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("v", [300, 5000])
@pytest.mark.parametrize("kw", SETTINGS)
def test_special_rows(kw, v, dev):
    x, u = special_rows(v)
    tok, lp = fm.kernels.sample_tokens(x.to(dev), u.to(dev), **kw)
    check(x, u, tok, lp, **kw)


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
def test_random_numbers_at_and_past_their_ends(dev):
    x = torch.tensor([[0.0, 0.0, 0.0, 0.0, -float("inf")]] * 9)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan")])
    tok, lp = fm.kernels.sample_tokens(x.to(dev), u.to(dev))
    assert tok.tolist() == [0, 1, 2, 3, 3, 3, 3, 0, 0]
    assert ((lp.cpu() + np.log(4.0)).abs() < 1e-6).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
def test_settings_per_row(dev):
    x, u = zipf(10, 700, 3)
    inf, nan = float("inf"), float("nan")
    temp = torch.tensor([1.0, 0.0, 0.5, -1.0, inf, nan, 2.0, 1e-30, 3e38, 1.0])
    top_k = torch.tensor([0, 5, -3, 4, 4, 4, 2 ** 40, 9, 3, 10])
    top_p = torch.tensor([0.9, 1.0, nan, 0.5, 0.5, 0.5, 2.0, 0.3, -1.0, 0.6])
    min_p = torch.tensor([0.0, 0.1, nan, 0.0, 0.0, 0.0, -2.0, 0.0, 0.0, 7.0])
    kw = dict(temperature=temp, top_k=top_k, top_p=top_p, min_p=min_p)
    tok, lp = fm.kernels.sample_tokens(x.to(dev), u.to(dev), **{k: t.to(dev) for k, t in kw.items()})
    assert (tok[3:6] == -1).all() and lp[3:6].isnan().all()
    top_p = torch.where(top_p.isnan(), 1.0, top_p).clamp(min=0)
    min_p = torch.where(min_p.isnan(), 0.0, min_p)
    for i in (0, 1, 2, 6, 7, 8, 9):
        check_row(x[i].numpy(), u[i].item(), tok[i].item(), lp[i].item(), temp[i].item(), min(int(top_k[i]), 700),
                  top_p[i].item(), min_p[i].item())


def test_refusals():
    x, u = zipf(3, 20, 1)
    for a in [(x[:, :0], u), (x.long(), u), (x, u[:2]), (x, u.long()), (x, u.to("meta")), (torch.tensor(1.0), u)]:
        with pytest.raises(ValueError):
            fm.kernels.sample_tokens(*a)
    for kw in [dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1),
               dict(top_k=2.5), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=float("nan")),
               dict(top_k=torch.ones(3)), dict(top_p=torch.ones(3, dtype=torch.int64)), dict(temperature=torch.ones(2)),
               dict(min_p=torch.ones(3, device="meta"))]:
        with pytest.raises(ValueError):
            fm.kernels.sample_tokens(x, u, **kw)
    t, lp = fm.kernels.sample_tokens(x[:0], u[:0], top_p=0.5)
    assert t.shape == (0,) and lp.shape == (0,)
    t, lp = fm.kernels.sample_tokens(x[0], u[0], top_p=0.5)
    assert t.shape == () and lp.shape == ()


def test_entry_point_validation():
    lib = _hip.lib()

    def f(n=2, v=8, dt=2, p=None):
        return lib.fm_sample(p, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, None, n, v, dt, None)
    assert f() == 1 and f(n=-1) == 1 and f(v=0) == 1 and f(dt=7) == 1 and f(v=2 ** 20 + 1) == 2 and f(n=2 ** 31) == 2
    assert f(n=2 ** 22) == 2
    assert f(n=0) == 0 and f(p=ctypes.c_void_p(65), dt=0) == 1


# ------------------------------------------------------------------ GPU
@gpu
@pytest.mark.parametrize("kw", SETTINGS)
@pytest.mark.parametrize("n,v,dt", [(7, 1, F32), (5, 7, BF16), (9, 64, F16), (6, 1000, F32), (4, 2049, BF16), (6, 8192, F32),
                                    (5, 32000, BF16), (3, 50257, F32), (3, 50257, F16), (3, 128256, BF16)])
def test_tokens_on_gpu(n, v, dt, kw):
    x, u = zipf(n, v, n + v, dt)
    fm.kernels.reset_stats()
    tok, lp = fm.kernels.sample_tokens(x.to(DEV), u.to(DEV), **kw)
    assert fm.kernels.stats() == {"fast": 1, "fallback": 0, "reasons": {}}
    check(x, u, tok, lp, **kw)


@gpu
def test_many_rows_of_every_steepness():
    x, u = zipf(400, 5003, 77, F32)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=30, top_p=0.9), dict(min_p=0.01)):
        tok, lp = fm.kernels.sample_tokens(x.to(DEV), u.to(DEV), **kw)
        check(x, u, tok, lp, **kw)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_cuts_inside_long_runs_of_equal_values(dt):
    # more equal values at the cut than a list holds: the search over the bits of the value, and the
    # cut in index order among them
    n, v = 6, 40000
    g = torch.Generator().manual_seed(4)
    x = torch.randint(0, 4, (n, v), generator=g).float()
    x[1] = 2.0
    x[2, :30] = 9.0
    x[3] = torch.where(torch.rand(v, generator=g) < 0.5, 1.0, -float("inf"))
    x[4, 100] = 5000.0
    x[5] = torch.randint(-2, 1, (v,), generator=g).float() * 0.001
    x = x.to(dt)
    u = torch.tensor([.123, .456, .789, .31, .77, .999])
    for kw in (dict(top_k=7), dict(top_k=5000), dict(top_k=25000, top_p=0.7), dict(top_p=0.37), dict(top_p=0.91, min_p=0.3),
               dict(top_k=35, top_p=0.9999), dict(temperature=5.0, top_p=0.5)):
        tok, lp = fm.kernels.sample_tokens(x.to(DEV), u.to(DEV), **kw)
        check(x, u, tok, lp, **kw)


@gpu
def test_shapes_strides_and_alignment():
    x, u = zipf(12, 1003, 8, BF16)
    xd, ud = x.to(DEV), u.to(DEV)
    want = fm.kernels.sample_tokens(xd, ud, top_p=0.8)
    check(x, u, *want, top_p=0.8)
    flat = torch.full((12 * 1003 + 9,), float("nan"), device=DEV, dtype=BF16)
    for off in (1, 3, 8):
        flat[off:off + 12 * 1003].view(12, 1003).copy_(xd)
        got = fm.kernels.sample_tokens(flat[off:off + 12 * 1003].view(12, 1003), ud, top_p=0.8)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        flat.fill_(float("nan"))
    wide = torch.full((12, 1100), float("nan"), device=DEV, dtype=BF16)
    wide[:, 20:1023] = xd
    for y, w in ((wide[:, 20:1023], ud), (xd.view(3, 4, 1003), ud.view(3, 4)), (xd.t().contiguous().t(), ud),
                 (xd, ud.repeat_interleave(2)[::2])):
        got = fm.kernels.sample_tokens(y, w, top_p=torch.full(w.shape, 0.8, device=DEV))
        assert torch.equal(got[0].view(-1), want[0]) and torch.equal(got[1].view(-1), want[1])


@gpu
def test_a_row_does_not_depend_on_its_batch_stream_or_replay():
    x, u = zipf(300, 32000, 9, BF16)
    xd, ud = x.to(DEV), u.to(DEV)
    kws = (dict(), dict(top_p=0.9), dict(top_k=50, top_p=0.9), dict(min_p=0.02), dict(top_k=3000))
    want = [fm.kernels.sample_tokens(xd, ud, **kw) for kw in kws]
    for (tok, lp), kw in zip(want, kws):
        for lo, hi in ((0, 1), (5, 6), (100, 117), (1, 300)):
            t, l = fm.kernels.sample_tokens(xd[lo:hi], ud[lo:hi], **kw)
            assert torch.equal(t, tok[lo:hi]) and torch.equal(l, lp[lo:hi]), (kw, lo, hi)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [fm.kernels.sample_tokens(xd, ud, **kw) for kw in kws]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    xs, us = xd[:16].clone(), ud[:16].clone()
    with torch.cuda.graph(graph):
        outs = [fm.kernels.sample_tokens(xs, us, **kw) for kw in kws]
    for a, b in zip(want, others):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for lo in (0, 40, 0):
        xs.copy_(xd[lo:lo + 16])
        us.copy_(ud[lo:lo + 16])
        graph.replay()
        torch.cuda.synchronize()
        for (t, l), (tok, lp) in zip(outs, want):
            assert torch.equal(t, tok[lo:lo + 16]) and torch.equal(l, lp[lo:lo + 16])


@gpu
@pytest.mark.parametrize("kw", [dict(top_p=0.5), dict(top_p=0.99), dict(top_p=0.9999), dict(top_k=2000), dict(top_k=30000),
                                dict(top_k=6000, top_p=0.9), dict(top_k=900, top_p=0.99), dict(min_p=0.3), dict(min_p=1e-6),
                                dict(top_p=0.9, min_p=0.2), dict(top_k=50, min_p=0.9), dict(temperature=0.3, top_p=0.95)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_flat_rows_and_long_lists(dt, kw):
    # steps with thousands of different values, lists that overflow, cuts deep in the row, candidates side
    # by side at one end, rows with fewer values left than top_k asks for
    g = torch.Generator().manual_seed(12)
    v = 60001
    x = torch.stack([0.02 * torch.randn(v, generator=g), 0.5 * torch.randn(v, generator=g) + 14, 3 * torch.randn(v, generator=g),
                     torch.linspace(9, -9, v), torch.linspace(-3, 3, v).square(), torch.full((v,), -float("inf"))])
    x[5, 11::29] = torch.randn(len(range(11, v, 29)), generator=g)
    x = x.to(dt)
    u = torch.tensor([.41, .97, .03, .55, .5, .76])
    tok, lp = fm.kernels.sample_tokens(x.to(DEV), u.to(DEV), **kw)
    check(x, u, tok, lp, **kw)


@gpu
@pytest.mark.parametrize("n", [2, 300])
@pytest.mark.parametrize("dt,v", [(F32, 2 ** 20), (BF16, 2 ** 20), (F16, 2 ** 20 - 3)])
def test_the_longest_rows(dt, v, n):
    # one element off a 16-byte border, more rows than compute units among the counts; the rows past the
    # second repeat it
    x, u = zipf(2, v, 21, dt)
    flat = torch.full((n * v + 1,), float("nan"), device=DEV, dtype=dt)
    xd = flat[1:].view(n, v)
    xd[0], xd[1:] = x[0].to(DEV), x[1].to(DEV)
    ud = torch.cat([u[:1], u[1:].expand(n - 1)]).to(DEV)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=40), dict(top_k=100000, top_p=0.999), dict(min_p=0.001)):
        tok, lp = fm.kernels.sample_tokens(xd, ud, **kw)
        assert (tok[1:] == tok[1]).all() and (lp[1:] == lp[1]).all()
        check(x, u, tok[:2], lp[:2], **kw)


@gpu
def test_more_rows_than_a_launch_takes():
    n, v = 2 ** 22, 3
    x = torch.tensor([[0.0, 3.0, 1.0]], device=DEV).repeat(n, 1)
    u = torch.full((n,), 0.5, device=DEV)
    for m in (n - 1, n):
        tok, lp = fm.kernels.sample_tokens(x[:m], u[:m], top_k=1)
        assert tok.shape == (m,) and (tok == 1).all() and (lp == 0).all()


@gpu
def test_rows_past_two_to_the_31_elements():
    n, v = 16800, 128256
    assert n * v > 2 ** 31
    x, u = zipf(64, v, 31, BF16)
    xd = x.to(DEV).repeat((n + 63) // 64, 1)[:n]
    ud = u.to(DEV).repeat((n + 63) // 64)[:n]
    for kw in (dict(top_k=50, top_p=0.9), dict(top_p=0.9)):
        tok, lp = fm.kernels.sample_tokens(xd, ud, **kw)
        want = fm.kernels.sample_tokens(xd[:64], ud[:64], **kw)
        rows = torch.arange(n, device=DEV) % 64
        assert torch.equal(tok, want[0][rows]) and torch.equal(lp, want[1][rows])


@gpu
def test_sampled_listed_and_trained_on():
    # on-policy distillation: the student's token, the teacher's list at that position, the loss
    g = torch.Generator().manual_seed(2)
    n, v, k = 33, 4001, 16
    student = (2 * torch.randn(n, v, generator=g)).to(BF16)
    teacher = (2 * torch.randn(n, v, generator=g)).to(BF16)
    u = torch.rand(n, generator=g)
    sd, td = student.to(DEV).requires_grad_(True), teacher.to(DEV)
    tok, lp = fm.kernels.sample_tokens(sd, u.to(DEV), temperature=0.9, top_p=0.95)
    assert not tok.requires_grad and not lp.requires_grad
    check(student, u, tok, lp, temperature=0.9, top_p=0.95)
    vals, idx = fm.kernels.topk(td, k)
    lse = torch.logsumexp(td.float(), -1)
    loss = fm.kernels.kl_div_topk(sd, idx, vals, teacher_lse=lse, tail="bucket")
    loss.backward()
    ref, grad, size, _ = O.kl_topk(student, idx.cpu(), vals.cpu(), lse.cpu(), False, "bucket")
    assert abs(loss.item() - ref.mean().item()) <= 1e-5 * abs(ref.mean().item())
    bound = 2.0 ** -8 * grad.abs() / n + 300 * 2.0 ** -24 * size / n + 1e-38
    assert ((sd.grad.double().cpu() - grad / n).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("dt,v", [(F32, 32000), (BF16, 32000), (F16, 50257), (BF16, 9001)])
def test_a_row_alone_is_the_row_among_many(dt, v):
    """Token and log-probability are the same bits with more rows than compute units and with fewer,
    where other workgroup sizes run. Half of the rows are one sequence of logits twice over, drawn at
    u = 1/2: in exact arithmetic the border lies between the two, so any difference in the order of the
    sums, or in how a weight is rounded, decides."""
    n = 300
    g = torch.Generator().manual_seed(v)
    half = v // 2
    x = torch.empty(n, v)
    a = torch.randn(n, half, generator=g) * (0.05 + 3 * torch.rand(n, 1, generator=g))
    x[:, :half], x[:, half:2 * half] = a, a
    if v % 2:
        x[:, -1] = -float("inf")
    x[1::2], u = zipf(n // 2, v, v + 1)[0], torch.full((n,), 0.5)
    u[1::2] = torch.rand(n // 2, generator=g)
    x = x.to(dt)
    xd, ud = x.to(DEV), u.to(DEV)
    for kw in (dict(), dict(temperature=0.7), dict(min_p=1e-3), dict(min_p=1e-5), dict(min_p=0.2), dict(top_k=600),
               dict(top_k=900), dict(top_k=3000), dict(top_k=5000, top_p=0.999), dict(top_p=0.5), dict(top_p=0.95),
               dict(top_p=0.9999), dict(top_k=3000, min_p=1e-4), dict(top_p=0.99, min_p=1e-3)):
        tok, lp = fm.kernels.sample_tokens(xd, ud, **kw)
        for lo in range(0, n, 50):
            t, l = fm.kernels.sample_tokens(xd[lo:lo + 50], ud[lo:lo + 50], **kw)
            assert torch.equal(t, tok[lo:lo + 50]) and torch.equal(l, lp[lo:lo + 50]), (kw, lo)


@gpu
def test_any_number_of_rows_and_elements_runs_on_the_kernel():
    n, v = 2 ** 22 + 5, 3
    fm.kernels.reset_stats()
    x = torch.tensor([[0.0, 3.0, 1.0]], device=DEV).repeat(n, 1)
    u = torch.rand(n, device=DEV)
    temp = 0.5 + torch.rand(n, device=DEV)
    tok, lp = fm.kernels.sample_tokens(x, u, temperature=temp, top_k=2)
    assert tok.shape == (n,) and lp.shape == (n,)
    for lo in (0, 2 ** 21, n - 7):
        t, l = fm.kernels.sample_tokens(x[lo:lo + 7], u[lo:lo + 7], temperature=temp[lo:lo + 7], top_k=2)
        assert torch.equal(t, tok[lo:lo + 7]) and torch.equal(l, lp[lo:lo + 7])
    # 2^33 elements and more: 17 GB of logits
    n, v = 67000, 128256
    assert n * v > 2 ** 33
    x, u = zipf(64, v, 33, BF16)
    xd = x.to(DEV).repeat((n + 63) // 64, 1)[:n]
    ud = u.to(DEV).repeat((n + 63) // 64)[:n]
    tok, lp = fm.kernels.sample_tokens(xd, ud, top_k=50, top_p=0.9)
    want = fm.kernels.sample_tokens(xd[:64], ud[:64], top_k=50, top_p=0.9)
    rows = torch.arange(n, device=DEV) % 64
    assert torch.equal(tok, want[0][rows]) and torch.equal(lp, want[1][rows])
    assert fm.kernels.stats()["fallback"] == 0


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("kind", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_top_k_of_every_integer_type(kind, dev):
    x, u = zipf(5, 700, 12)
    top_k = torch.tensor([0, 1, 7, 100, 127])
    want = fm.kernels.sample_tokens(x.to(dev), u.to(dev), top_k=top_k.to(dev))
    got = fm.kernels.sample_tokens(x.to(dev), u.to(dev), top_k=top_k.to(kind).to(dev))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for i in range(5):
        check_row(x[i].numpy(), u[i].item(), got[0][i].item(), got[1][i].item(), top_k=int(top_k[i]))
    if kind == torch.int64:       # past 32 bits: everything stays
        high = torch.tensor([2 ** 32 + 5, 2 ** 40, 2 ** 31, 2 ** 63 - 1, 700], device=dev)
        off = fm.kernels.sample_tokens(x.to(dev), u.to(dev))
        for t in (high, high.to(torch.uint64)):
            assert torch.equal(fm.kernels.sample_tokens(x.to(dev), u.to(dev), top_k=t)[0], off[0])
    if kind != torch.uint8:       # negative: off, also below the least of 32 bits
        low = torch.full((5,), torch.iinfo(kind).min, dtype=kind, device=dev)
        off = fm.kernels.sample_tokens(x.to(dev), u.to(dev))
        assert torch.equal(fm.kernels.sample_tokens(x.to(dev), u.to(dev), top_k=low)[0], off[0])


def test_numbers_that_32_bits_do_not_hold_are_refused():
    x, u = zipf(2, 20, 1)
    for kw in [dict(temperature=1e39), dict(temperature=3.5e38), dict(top_k=float("inf")), dict(top_k=float("nan"))]:
        with pytest.raises(ValueError):
            fm.kernels.sample_tokens(x, u, **kw)
    a = fm.kernels.sample_tokens(x, u, temperature=torch.finfo(F32).max, top_k=2 ** 70)
    b = fm.kernels.sample_tokens(x * 0, u)
    assert torch.equal(a[0], b[0])
