"""The code-score operators on the GPU against plain 64-bit evaluations of their definitions.

Tolerances come from the operations: U = 2^-24 is half a step of fp32; a chain of n fp32 operations errs by at most n U times the sum of
the terms' magnitudes.  Drawn codes, counts and arguments of maxima are integers and have to be equal."""
import numpy as np
import pytest
import torch

import lbm_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def f64(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------------------------------------------------- code_logits
def logits64(x, e, T, ee=None):
    n = (e * e).sum(1) if ee is None else ee
    return (2 * x @ e.T - n) / T


def logits_tol(x, e, T, ee=None):
    D = x.shape[1]
    n = (e * e).sum(1) if ee is None else np.abs(ee)
    mag = 2 * np.abs(x) @ np.abs(e).T + n           # a chain of D products each, then the sum, the scale and its rounding
    return U * (D + 8) * mag / T + 1e-37


@pytest.mark.parametrize("N,D,K", [(1, 1, 1), (1, 256, 512), (2, 3, 5), (63, 8, 65), (64, 32, 64), (129, 33, 127), (375, 256, 413), (1000, 100, 70),
                                   (4100, 256, 1030), (5, 257, 8192), (40, 64, 7001), (1, 256, 8192)])
@pytest.mark.parametrize("T", [1.0, 0.07])
def test_logits_and_gradients(N, D, K, T):
    g = gen(N * 7 + D * 3 + K)
    x, e, w = torch.randn((N, D), generator=g), torch.randn((K, D), generator=g), torch.randn((N, K), generator=g)
    xd, ed = x.to(DEV).requires_grad_(), e.to(DEV).requires_grad_()
    s = lbm_amd.code_logits(xd, ed, temperature=T)
    assert s.shape == (N, K) and s.dtype == torch.float32
    x64, e64, w64 = f64(x), f64(e), f64(w)
    assert (np.abs(f64(s) - logits64(x64, e64, T)) <= logits_tol(x64, e64, T)).all()
    dx, de = torch.autograd.grad(s, (xd, ed), w.to(DEV))
    want_dx = 2 / T * w64 @ e64
    want_de = 2 / T * (w64.T @ x64 - w64.sum(0)[:, None] * e64)
    assert (np.abs(f64(dx) - want_dx) <= U * (K + 8) * 2 / T * (np.abs(w64) @ np.abs(e64)) + 1e-37).all()
    mag = np.abs(w64).T @ np.abs(x64) + np.abs(w64).sum(0)[:, None] * np.abs(e64)
    assert (np.abs(f64(de) - want_de) <= U * (N + 16) * 2 / T * mag + 1e-37).all()
    # one of the two gradients alone is the same numbers; a second run is the same bits
    (dx1,) = torch.autograd.grad(lbm_amd.code_logits(xd, ed.detach(), temperature=T), xd, w.to(DEV))
    (de1,) = torch.autograd.grad(lbm_amd.code_logits(xd.detach(), ed, temperature=T), ed, w.to(DEV))
    assert torch.equal(dx1, dx) and torch.equal(de1, de)


def test_logits_gradients_against_differences():
    """Central differences of sum(w * s) in 64 bits through the fp32 kernel: s is quadratic, so the difference has no step error and only
    the scores' rounding counts: at most tol(s) * sum|w| / step per entry."""
    g = gen(3)
    N, D, K, T, step = 6, 5, 7, 0.5, 0.25
    x, e, w = torch.randn((N, D), generator=g), torch.randn((K, D), generator=g), torch.randn((N, K), generator=g)
    xd, ed = x.to(DEV).requires_grad_(), e.to(DEV).requires_grad_()
    dx, de = torch.autograd.grad(lbm_amd.code_logits(xd, ed, T), (xd, ed), w.to(DEV))

    def loss(a, b):
        return float((f64(lbm_amd.code_logits(a.to(DEV), b.to(DEV), T)) * f64(w)).sum())
    big = (np.abs(f64(x)).max() + step), (np.abs(f64(e)).max() + step)
    tol = logits_tol(np.full((1, D), big[0]), np.full((1, D), big[1]), T)[0, 0] * np.abs(f64(w)).sum() / step + 1e-6
    for t, grad, f in ((x, dx, lambda p: loss(p, e)), (e, de, lambda p: loss(x, p))):
        for i in range(t.shape[0]):
            for d in range(t.shape[1]):
                a, b = t.clone(), t.clone()
                a[i, d] += step
                b[i, d] -= step
                width = float(a[i, d].double() - b[i, d].double())
                assert abs((f(a) - f(b)) / width - float(grad[i, d])) <= tol


@pytest.mark.parametrize("B,S,D,K", [(1, 1, 4, 3), (3, 5, 16, 33), (7, 375, 256, 512), (2, 130, 20, 100)])
def test_logits_channel_major(B, S, D, K):
    from lbm_amd.quantizer import pitched_empty
    g = gen(B + S)
    z, e = torch.randn((B, D, S), generator=g), torch.randn((K, D), generator=g)
    zp = pitched_empty(B, D, S, DEV)
    zp.copy_(z)
    got = lbm_amd.code_logits(zp, e.to(DEV), 0.5, channel_major=True)
    rows = z.permute(0, 2, 1).reshape(-1, D)
    assert (np.abs(f64(got) - logits64(f64(rows), f64(e), 0.5)) <= logits_tol(f64(rows), f64(e), 0.5)).all()
    assert torch.equal(got, lbm_amd.code_logits(z.to(DEV), e.to(DEV), 0.5, channel_major=True))
    zd = z.to(DEV).requires_grad_()
    w = torch.randn((B * S, K), generator=g)
    (dz,) = torch.autograd.grad(lbm_amd.code_logits(zd, e.to(DEV), 0.5, channel_major=True), zd, w.to(DEV))
    want = (4 * f64(w) @ f64(e)).reshape(B, S, D).transpose(0, 2, 1)
    mag = (4 * np.abs(f64(w)) @ np.abs(f64(e))).reshape(B, S, D).transpose(0, 2, 1)
    assert (np.abs(f64(dz) - want) <= U * (K + 8) * mag).all()


def test_logits_strides_offsets_and_given_norms():
    g = gen(11)
    base = torch.randn((40, 77), generator=g).to(DEV)
    e = torch.randn((90, 64), generator=g).to(DEV)
    for x in (base[:, 3:67], base[::2, 5:69], base.t()[:64, :].t(), torch.randn((64,), generator=g).to(DEV).expand(5, 64)):
        for cb in (e, e[1::2], e.flatten()[1:1 + 33 * 64].view(33, 64)):      # the last: not 16-byte aligned
            s = lbm_amd.code_logits(x, cb)
            assert (np.abs(f64(s) - logits64(f64(x), f64(cb), 1.0)) <= logits_tol(f64(x), f64(cb), 1.0)).all()
    ee = torch.randn((90,), generator=g).to(DEV)
    x = base[:, 3:67].contiguous().requires_grad_()
    ed = e.clone().requires_grad_()
    s = lbm_amd.code_logits(x, ed, 0.5, e_sqnorm=ee)
    assert (np.abs(f64(s) - logits64(f64(x), f64(e), 0.5, f64(ee))) <= logits_tol(f64(x), f64(e), 0.5, f64(ee))).all()
    w = torch.randn((40, 90), generator=g).to(DEV)
    dx, de = torch.autograd.grad(s, (x, ed), w)
    assert (np.abs(f64(de) - 4 * f64(w).T @ f64(x)) <= U * (40 + 16) * 4 * np.abs(f64(w)).T @ np.abs(f64(x))).all()
    # a broadcast gradient (stride 0), and a codebook in half precision whose gradient comes back in its type
    (d1,) = torch.autograd.grad(lbm_amd.code_logits(x, e).sum(), x)
    want = np.broadcast_to(2 * f64(e).sum(0), (40, 64))
    assert (np.abs(f64(d1) - want) <= U * 98 * 2 * np.abs(f64(e)).sum(0)).all()
    eh = e.half().requires_grad_()
    (dh,) = torch.autograd.grad(lbm_amd.code_logits(x.detach(), eh), eh, w)
    assert dh.dtype == torch.float16
    assert lbm_amd.code_logits(x.detach()[:0], e).shape == (0, 90)


# --------------------------------------------------------------------------------------------------------------- balance
def balance64(s, codes, keep, gl, gm):
    """(loss, counts, mean, ds) and the bound of each one's error in fp32 before the scores' type rounds ds."""
    N, K = s.shape
    on = (np.ones(N, bool) if keep is None else keep.copy())
    on[on] &= (s[on] > -np.inf).any(1)
    p, tp = np.zeros((N, K)), np.zeros((N, K))
    for n in np.nonzero(on)[0]:
        d = s[n] - s[n].max()
        w = np.exp(d)
        p[n] = w / w.sum()
        dist = np.where(np.isfinite(d), np.abs(d), 0.0)
        # the difference rounds (|d| U), the exponential errs by 4 U, the sum and its reciprocal by 48 U and the weights' own errors
        tp[n] = U * p[n] * (dist + (p[n] * dist).sum() + 64)
    M = int(on.sum())
    if codes is None:
        picks = [int(np.nonzero(s[n] == s[n].max())[0][0]) for n in np.nonzero(on)[0]]
    else:
        picks = codes[on].ravel()
        picks = picks[(picks >= 0) & (picks < K)]
    counts = np.bincount(np.asarray(picks, np.int64), minlength=K)
    C = counts.sum()
    f = counts / C if C else np.zeros(K)
    mean = p.sum(0) / M if M else np.zeros(K)
    tmean = tp.sum(0) / M + U * (N + 16) * mean if M else np.zeros(K)    # at most N additions into one sum
    loss, tloss = K * (f * mean).sum(), K * (f * tmean).sum() + 4 * U * K * (f * mean).sum()
    a = gl * K * f + gm
    ds, tds = np.zeros((N, K)), np.zeros((N, K))
    for n in np.nonzero(on)[0]:
        ref = a[s[n] == s[n].max()].max()
        b = a - ref
        tb = U * (np.abs(a) + abs(ref) + np.abs(b))
        t, tt = (p[n] * b).sum(), (p[n] * tb + tp[n] * np.abs(b) + 48 * U * p[n] * np.abs(b)).sum()
        ds[n] = p[n] * (b - t) / M
        tds[n] = (tp[n] * np.abs(b - t) + p[n] * (tb + tt) + 4 * U * p[n] * np.abs(b - t)) / M
    return loss, counts, mean, ds, tloss, tmean, tds


def check_balance(s, codes, keep, seed=0, gl=0.3):
    N, K = s.reshape(-1, s.shape[-1]).shape
    gm = torch.randn((K,), generator=gen(seed)) * 0.05
    sd = s.to(DEV).requires_grad_()
    loss, counts, mean = lbm_amd.code_balance_loss(sd, None if codes is None else codes.to(DEV), keep=None if keep is None else keep.to(DEV))
    assert loss.shape == () and counts.shape == (K,) and mean.shape == (K,) and counts.dtype == torch.int64
    (ds,) = torch.autograd.grad((loss, mean), (sd,), (torch.tensor(gl, device=DEV), gm.to(DEV)))
    assert ds.dtype == s.dtype and ds.shape == s.shape
    c = None if codes is None else codes.reshape(N, -1).numpy()
    k = None if keep is None else keep.reshape(-1).numpy()
    # the upstream gradients as the kernel is given them: fp32
    wl, wc, wm, wds, tl, tm, tds = balance64(f64(s).reshape(N, K), c, k, float(np.float32(gl)), f64(gm))
    assert np.array_equal(counts.cpu().numpy(), wc)
    assert (np.abs(f64(mean) - wm) <= tm + 1e-37).all(), np.abs(f64(mean) - wm).max()
    assert abs(float(loss.detach()) - wl) <= tl + 1e-37
    fi = torch.finfo(s.dtype)
    tds = tds + (0 if s.dtype == torch.float32 else np.abs(wds) * fi.eps / 2 + fi.smallest_normal * fi.eps)   # the type's rounding
    err = np.abs(f64(ds).reshape(N, K) - wds)
    assert (err <= tds + 1e-37).all(), (err - tds).max()
    return loss, counts, mean, ds


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,K", [(1, 1), (1, 512), (3, 2), (5, 61), (64, 256), (37, 257), (200, 512), (130, 1000), (33, 2048), (21, 2052), (9, 4097),
                                 (17, 8192), (6, 8191)])
def test_balance_sizes_and_types(kind, N, K):
    g = gen(N + K)
    s = (torch.randn((N, K), generator=g) * 3).to(TYPES[kind])
    check_balance(s, torch.randint(0, K, (N,), generator=g), None)
    check_balance(s, None, torch.rand((N,), generator=g) < 0.6)
    check_balance(s, torch.randint(-1, K + 1, (N, 3), generator=g), torch.rand((N,), generator=g) < 0.8)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("K", (1, 2, 5, 8, 9, 17, 32, 33, 64, 65, 100, 128, 129))
def test_balance_rows_that_share_a_wave(kind, K):
    g = gen(1000 + K)
    s = (torch.randn((1237, K), generator=g) * 3).to(TYPES[kind])
    s[5::7, : K // 2] = float("-inf")
    s[11::13] = float("-inf")                     # rows that end early beside rows that do not
    check_balance(s, None, torch.rand((1237,), generator=g) < 0.7)
    check_balance(s[:1200:3], torch.randint(-1, K, (400, 40), generator=g), None)      # more picks than lanes


@pytest.mark.parametrize("K", (5, 100, 600, 1500, 3001, 8192))
@pytest.mark.parametrize("offset", (9e5, -9e5, 999_000.0, 3e6, 3e33))
def test_balance_scores_far_from_zero(offset, K):
    # p depends on differences alone, which are exact here (scores of one binade; at 3e33 equal but for a code far below)
    s = (torch.randn((33, K), generator=gen(K)) * 3 + offset).float()
    s[:, 0] -= abs(offset) / 8
    check_balance(s, torch.arange(33) % K, None)
    check_balance(s, None, None)


def test_balance_many_rows():
    g = gen(5)
    s = torch.randn((30011, 96), generator=g) * 2
    codes = torch.randint(0, 96, (30011,), generator=g)
    a = check_balance(s, codes, torch.rand((30011,), generator=g) < 0.9)
    b = check_balance(s, codes, torch.rand((30011,), generator=gen(5)) < 2)      # every row
    c = check_balance(s, codes, None)
    for x, y in zip(b, c):
        assert torch.equal(x, y)                  # a mask that keeps all is no mask, bit for bit
    assert not torch.equal(a[1], b[1])


def test_balance_masks_and_extremes():
    g = gen(6)
    s = torch.randn((40, 70), generator=g)
    s[3] = float("-inf")                          # a row with nothing in it
    s[4, 1:] = float("-inf")                      # one code
    s[5] = torch.finfo(torch.float32).min         # all of them the type's lowest value: even
    s[6, 10:] = torch.finfo(torch.float32).min
    s[7] = 80.0 * s[7]                            # one probability near 1
    s[8, 5] = 300.0
    keep = torch.ones((40,), dtype=torch.bool)
    keep[9:12] = False
    s[9], s[10], s[11] = float("nan"), float("inf"), float("-inf")
    _, counts, _, ds = check_balance(s, None, keep)
    assert int(counts.sum()) == 36 and not ds[[3, 9, 10, 11]].any() and torch.isfinite(ds).all()
    _, counts, _, _ = check_balance(s, torch.arange(40) % 70, keep)
    assert counts[3] == 0 and counts[9] == 0 and int(counts.sum()) == 36
    # nothing counts at all: zeros, no NaN
    for k in (torch.zeros((40,), dtype=torch.bool), None):
        t = s if k is not None else torch.full((4, 70), float("-inf"))
        _, counts, mean, ds = check_balance(t, None, k)
        assert not counts.any() and not mean.any() and not ds.any()
    # no rows
    loss, counts, mean = lbm_amd.code_balance_loss(torch.zeros((0, 9), device=DEV, requires_grad=True))
    assert float(loss.detach()) == 0 and not counts.any() and not mean.any()
    # NaN in a row that counts is seen
    bad = torch.randn((3, 8), generator=g)
    bad[1, 2] = float("nan")
    assert torch.isnan(lbm_amd.code_balance_loss(bad.to(DEV))[0])
    assert torch.isnan(lbm_amd.code_balance_loss(torch.full((2, 8), float("nan"), device=DEV))[0])


def test_balance_even_and_collapsed_use():
    s = torch.zeros((64, 64))
    loss, counts, mean = lbm_amd.code_balance_loss(s.to(DEV), torch.arange(64).to(DEV))
    assert float(loss) == 1.0 and (counts == 1).all() and (mean == 1 / 64).all()
    s = torch.full((64, 64), -200.0)
    s[:, 5] = 200.0
    loss, counts, _ = lbm_amd.code_balance_loss(s.to(DEV))
    assert float(loss) == 64.0 and int(counts[5]) == 64


def test_balance_strides_shapes_and_ties():
    g = gen(8)
    base = torch.randn((20, 200), generator=g)
    for s in (base[:, 3:103], base[::3, :100], base.t()[:100].t(), base[:1, :64].expand(20, 64)):
        check_balance(s, None, None)
    s = torch.randn((2, 3, 5, 24), generator=g)
    check_balance(s, torch.randint(0, 24, (2, 3, 5), generator=g), torch.rand((2, 3, 5), generator=g) < 0.7)
    check_balance(s, torch.randint(0, 24, (2, 3, 5, 2), generator=g).to(torch.int32), None)
    t = torch.randint(0, 3, (50, 300), generator=g).float()       # many equal best scores: the lowest index counts
    check_balance(t, None, None)
    check_balance(t.bfloat16(), None, None)


def test_balance_gradient_of_single_outputs_and_of_differences():
    g = gen(9)
    s = torch.randn((7, 11), generator=g)
    codes = torch.randint(0, 11, (7,), generator=g).to(DEV)
    sd = s.to(DEV).requires_grad_()
    loss, _, mean = lbm_amd.code_balance_loss(sd, codes)
    d_loss = torch.autograd.grad(loss, sd, retain_graph=True)[0]
    gm = torch.randn((11,), generator=g).to(DEV)
    d_mean = torch.autograd.grad(mean, sd, gm)[0]

    def value(t):
        p = torch.softmax(t, 1).mean(0)
        f = torch.bincount(codes.cpu(), minlength=11).double() / 7
        return float(11 * (f * p).sum()), float((p * gm.cpu().double()).sum())
    h = 1e-5
    for n in range(7):
        for k in range(11):
            a, b = s.double(), s.double()
            a[n, k] += h
            b[n, k] -= h
            va, vb = value(a), value(b)
            # third derivatives are below 11 here, so the step adds at most 11 h^2; the kernel's own error is below 1e-6
            assert abs((va[0] - vb[0]) / (2 * h) - float(d_loss[n, k])) <= 2e-6
            assert abs((va[1] - vb[1]) / (2 * h) - float(d_mean[n, k])) <= 2e-6


# -------------------------------------------------------------------------------------------------------------- sampling
def sample64(s, u, T, top_k, top_p, min_p, allowed=None):
    N, K = s.shape
    out = np.empty(N, np.int64)
    for n in range(N):
        v = np.where(np.isnan(s[n]), -np.inf, s[n])
        if allowed is not None:
            v = np.where(allowed[n], v, -np.inf)
        m = v.max()
        if m == -np.inf:
            out[n] = -1
            continue
        if not T[n] > 0:
            out[n] = int(np.argmax(v))
            continue
        with np.errstate(invalid="ignore"):
            w = np.where(v == m, 1.0, np.where((v == -np.inf) | (m == np.inf), 0.0, np.exp((v - m) / T[n])))   # +inf takes all weight
        order = np.lexsort((np.arange(K), -v))
        if top_k[n] > 0:
            order = order[:top_k[n]]
        if top_p[n] < 1:
            ws = w[order]
            before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
            stay = before < top_p[n] * ws.sum()
            stay[0] = True
            order = order[stay]
        left = np.sort(order[(w[order] >= min(max(min_p[n], 0.0), 1.0)) & (w[order] > 0)])
        cum = np.cumsum(w[left])
        out[n] = left[min(int(np.searchsorted(cum, u[n] * cum[-1], side="right")), len(left) - 1)]
    return out


def check_sample(s, u, allowed=None, **kw):
    N, K = s.shape
    par = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **kw}
    got = lbm_amd.sample_codes(s.to(DEV), u.to(DEV), allowed=None if allowed is None else allowed.to(DEV),
                               **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in par.items()})
    col = {k: (v.double().numpy() if isinstance(v, torch.Tensor) else np.full(N, float(v))) for k, v in par.items()}
    a = None if allowed is None else np.broadcast_to(allowed.numpy().astype(bool), (N, K))
    want = sample64(f64(s), f64(u), col["temperature"], col["top_k"].astype(np.int64), col["top_p"], col["min_p"], a)
    got = got.cpu().numpy()
    bad = np.nonzero(got != want)[0]
    assert bad.size == 0, (bad[:5], got[bad[:5]], want[bad[:5]])
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(top_k=1), dict(top_k=7), dict(top_p=0.9), dict(top_p=0.0), dict(min_p=0.05),
            dict(min_p=1.0), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.02), dict(temperature=5.0, top_p=0.5, min_p=0.3),
            dict(temperature=1.5, top_k=5, top_p=0.99), dict(top_k=380), dict(top_k=1000), dict(temperature=3.0, top_p=0.999),
            dict(temperature=4.0, top_k=900, top_p=0.97, min_p=0.001)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,K", [(1, 1), (1, 512), (5, 2), (66, 61), (40, 256), (41, 258), (200, 512), (50, 1023), (30, 2048), (20, 2049), (17, 4100),
                                 (12, 8192), (7, 8191), (3, 70001)])
def test_sample_sizes_types_settings(kind, N, K):
    g = gen(N * 31 + K)
    s = (torch.randn((N, K), generator=g) * 3).to(TYPES[kind])
    u = torch.rand((N,), generator=g)
    for kw in SETTINGS:
        check_sample(s, u, **kw)


@pytest.mark.parametrize("K", [16, 300, 512, 3000])
def test_sample_ties(K):
    g = gen(K)
    u = torch.rand((60,), generator=g)
    for s in (torch.zeros((60, K)), torch.randint(0, 3, (60, K), generator=g).float(), torch.randint(-1, 1, (60, K), generator=g).float() * 1e30,
              -0.0 * torch.ones((60, K)) * torch.randint(-1, 2, (60, K), generator=g)):
        for kw in (dict(), dict(top_k=5), dict(top_p=0.5), dict(top_p=0.9, top_k=K // 2), dict(min_p=1.0), dict(temperature=0.0),
                   dict(temperature=2.0, top_k=K - 1, top_p=0.75, min_p=0.3)):
            check_sample(s, u, **kw)
            check_sample(s.bfloat16(), u, **kw)


def test_sample_u_at_the_ends_and_outside():
    g = gen(2)
    s = torch.randn((8, 100), generator=g)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, 0.5, 0.0, 1.0, 1e-30])
    for kw in (dict(), dict(top_k=3), dict(top_p=0.4, min_p=0.01)):
        check_sample(s, u, **kw)
    # rows whose weight lies in their first columns only, in the middle, at the end
    for K in (900, 5000, 150_000):
        s = torch.full((8, K), float("-inf"))
        s[:4, 5:300] = torch.randn((4, 295), generator=g)
        s[4:6, K // 2:K // 2 + 90] = torch.randn((2, 90), generator=g)
        s[6:, -700:] = torch.randn((2, 700), generator=g)
        s[::2, 700:] = torch.maximum(s[::2, 700:], torch.tensor(-2000.0))      # there, but without weight in 64 bits
        for kw in (dict(), dict(top_k=280, top_p=0.999), dict(top_p=0.4, min_p=0.01), dict(min_p=1e-4), dict(temperature=0.0)):
            check_sample(s, u, **kw)
    s = torch.randn((8, 100), generator=g)
    # numbers that are none of [0, 1): the last code that stayed for NaN, the first for negative ones
    got = lbm_amd.sample_codes(s[:2].to(DEV), torch.tensor([float("nan"), -1.0], device=DEV)).cpu()
    assert got.tolist() == [99, 0]


def test_sample_masks_and_extremes():
    g = gen(4)
    for K in (70, 600, 5000):
        s = torch.randn((14, K), generator=g)
        lo = torch.finfo(torch.float32).min
        s[0] = float("-inf")
        s[1, 3:] = float("-inf")
        s[2] = lo
        s[3, 1:] = lo
        s[4, 7] = float("inf")
        s[5, ::5] = float("inf")
        s[6, ::2] = float("nan")
        s[7] = float("nan")
        s[8] = torch.finfo(torch.float32).max
        s[9] = s[9] * 1e30
        s[10] = s[10] * 1e-40                     # denormal scores: all weights near 1
        s[11, :K - 1] = float("-inf")
        s[12] = torch.linspace(-800, 0, K)        # weights down to nothing in 64 bits
        u = torch.rand((14,), generator=g)
        for kw in SETTINGS + [dict(top_k=2, top_p=0.6), dict(temperature=float("inf")), dict(temperature=1e-30), dict(top_k=10 ** 9)]:
            got = check_sample(s, u, **kw)
            assert got[0] == -1 and got[7] == -1
            check_sample(s, u, allowed=torch.rand((K,), generator=g) < 0.5, **kw)
        check_sample(s, u, allowed=torch.rand((14, K), generator=g) < 0.3, top_k=4)
        assert (check_sample(s, u, allowed=torch.zeros((K,), dtype=torch.bool)) == -1).all()


@pytest.mark.parametrize("K", [60, 256, 511, 1000])
def test_sample_short_rows_of_every_shape(K):
    # borders that halving and cutting the range of scores do not find soon: clusters, outliers, scores spaced as powers
    g = gen(40 + K)
    base = torch.randn((K,), generator=g)
    s = torch.stack([
        -torch.exp(torch.linspace(-30, 6, K))[torch.randperm(K, generator=g)],      # dense at the best score
        torch.exp(torch.linspace(-30, 3, K))[torch.randperm(K, generator=g)],       # dense at the lowest
        torch.where(torch.arange(K) == 7, torch.tensor(-1e30), base * 1e-3),        # one far below the others
        torch.where(torch.arange(K) == 7, torch.tensor(40.0), base * 1e-3),         # one far above
        5.0 + torch.arange(K) % 3 * 2.0 ** -21,                                     # three neighbouring floats
        torch.where(torch.arange(K) % 2 == 0, torch.tensor(3e38), torch.tensor(-3e38)) * (1 + base.abs() * 1e-2).clamp(max=1.1),
        base * 1e-42,
        base.sign() * torch.exp(base * 3),
    ])
    u = torch.rand((8,), generator=g)
    for kw in SETTINGS + [dict(top_k=K // 2), dict(top_k=K - 1), dict(top_p=0.5), dict(top_p=0.999), dict(top_p=0.3, temperature=30.0),
                          dict(top_k=K // 3, top_p=0.7, temperature=5.0)]:
        check_sample(s, u, **kw)


@pytest.mark.parametrize("K", [2, 64, 512, 1024, 5000])
def test_sample_nucleus_round_the_best_code(K):
    # top-p's share of the total lies just below, at and above the best code's weight of 1
    s = torch.full((60, K), -300.0)
    g = gen(50 + K)
    at = torch.randint(0, K, (60,), generator=g)
    s[torch.arange(60), at] = 0.0
    second = (at + 1 + torch.randint(0, K - 1, (60,), generator=g)) % K
    s[torch.arange(60), second] = -3.0 * torch.rand((60,), generator=g)
    s[40:, : K // 2] = torch.maximum(s[40:, : K // 2], -4.0 - torch.rand((20, K // 2), generator=g))
    s[::7] += 17.0
    u = torch.rand((60,), generator=g)
    u[:20] = 0.999
    w = np.exp(f64(s) - f64(s).max(1, keepdims=True)).sum(1)
    for n in range(60):
        for d in (-1e-2, -1.1e-3, -9e-4, -1e-5, -1e-9, 1e-9, 1e-5, 1e-3):
            p = min((1.0 + d) / w[n], 1.0)
            check_sample(s[n:n + 1], u[n:n + 1], top_p=p)
            check_sample(s[n:n + 1], u[n:n + 1], top_p=p, top_k=2)
    check_sample(s, u, top_p=torch.from_numpy(1.0 / w).float())
    check_sample(s, u, top_k=torch.randint(0, 3, (60,), generator=g))


@pytest.mark.parametrize("K", [1500, 8192])
def test_sample_long_rows_of_every_shape(K):
    """Rows whose order or spread misleads a look at a few of their scores."""
    g = gen(K + 1)
    r = torch.arange(K).float()
    s = torch.stack([r / K * 20, -r / K * 20, torch.randn((K,), generator=g) * 1e-3, torch.randn((K,), generator=g) * 1e3,
                     torch.where(r % 16 == 3, torch.randn((K,), generator=g) + 30, torch.randn((K,), generator=g)),      # all good ones between
                     torch.where(r < K // 2, torch.zeros(K), torch.full((K,), float("-inf"))),
                     torch.where(r == K - 2, torch.full((K,), 900.0), torch.randn((K,), generator=g)),
                     torch.where(r >= K - 600, torch.full((K,), 5.0), torch.randn((K,), generator=g)),
                     torch.where(r % 100 == 7, torch.randn((K,), generator=g), torch.full((K,), float("-inf"))),
                     torch.where(r % 4 == 1, torch.full((K,), float("nan")), torch.randn((K,), generator=g))])
    for seed in range(3):
        u = torch.rand((len(s),), generator=gen(seed))
        for kw in SETTINGS:
            check_sample(s, u, **kw)
            check_sample(s.bfloat16(), u, **kw)


def test_sample_per_row_settings():
    g = gen(12)
    for N, K in ((300, 512), (60, 1500), (40, 8192), (65, 77)):
        s = torch.randn((N, K), generator=g) * 2
        u = torch.rand((N,), generator=g)
        t = torch.rand((N,), generator=g) * 2
        t[::7] = 0.0
        t[1], t[2] = -1.0, float("nan")
        k = torch.randint(-2, 2 * K, (N,), generator=g)
        k[::3] = torch.randint(1, 9, ((N + 2) // 3,), generator=g)
        p = torch.rand((N,), generator=g) * 1.2
        m = torch.rand((N,), generator=g) * 0.2 - 0.05
        check_sample(s, u, temperature=t, top_k=k, top_p=p, min_p=m)
        check_sample(s, u, temperature=t, top_p=0.8)
        check_sample(s.half(), u, top_k=k, min_p=m)


def test_sample_strides_shapes_hist():
    g = gen(14)
    base = torch.randn((30, 700), generator=g)
    u = torch.rand((30,), generator=g)
    for s in (base[:, 1:513], base[:, 4:516], base.t()[:300].t(), base[:1, :100].expand(30, 100), base[:, ::2]):
        check_sample(s, u, top_p=0.9)
        got = lbm_amd.sample_codes(s.to(DEV), u.to(DEV), top_p=0.9)      # .to() may have made it dense: the view on the device too
        wide = torch.zeros((30, 2 * s.shape[1]), device=DEV)
        view = wide[:, 1:1 + s.shape[1]]
        view.copy_(s)
        assert torch.equal(lbm_amd.sample_codes(view, u.to(DEV), top_p=0.9), got)
    s3 = base[:, :512].reshape(5, 6, 512).to(DEV)
    hist = torch.full((512,), 3, dtype=torch.int64, device=DEV)
    s3[0, 0] = float("-inf")
    got = lbm_amd.sample_codes(s3, u.reshape(5, 6).to(DEV), top_k=9, hist=hist)
    assert got.shape == (5, 6) and int(got[0, 0]) == -1
    want = np.bincount(got.cpu().numpy().ravel()[1:], minlength=512) + 3
    assert np.array_equal(hist.cpu().numpy(), want)
    one = lbm_amd.sample_codes(s3[1, 1], u[0].to(DEV))
    assert one.shape == () and int(one) == int(check_sample(s3[1, 1].cpu()[None], u[:1])[0])
    assert lbm_amd.sample_codes(s3[:0], u.reshape(5, 6)[:0].to(DEV)).shape == (0, 6)


def test_sample_frequencies():
    """Codes come up as often as their weights say: 200 000 draws of one row, every count within 6 standard deviations."""
    g = gen(20)
    s = torch.randn((1, 50), generator=g)
    n = 200_000
    u = torch.rand((n,), generator=g)
    got = lbm_amd.sample_codes(s.expand(n, 50).to(DEV), u.to(DEV), temperature=0.8, top_k=20)
    w = np.exp(f64(s)[0] / 0.8)
    w[np.argsort(-w)[20:]] = 0
    p = w / w.sum()
    c = np.bincount(got.cpu().numpy(), minlength=50)
    assert (np.abs(c - n * p) <= 6 * np.sqrt(n * p * (1 - p)) + 1e-9).all()


# --------------------------------------------------------------------------------------------------- together, streams, graphs
def test_offsets_past_32_bits():
    """Rows whose scores lie beyond 2^31 elements: the last ones answer as the same rows alone."""
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 20 GB of device memory")
    N, K = 270_000, 8192                          # 2.2e9 scores in bf16
    s = torch.empty((N, K), dtype=torch.bfloat16, device=DEV)
    s.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    u = torch.rand((N,), device=DEV)
    got = lbm_amd.sample_codes(s, u, top_p=0.9)
    assert torch.equal(got[-50:], lbm_amd.sample_codes(s[-50:].clone(), u[-50:], top_p=0.9))
    keep = torch.zeros((N,), dtype=torch.bool, device=DEV)
    keep[-50:] = True
    a = lbm_amd.code_balance_loss(s, keep=keep)
    b = lbm_amd.code_balance_loss(s[-50:].clone())
    assert torch.equal(a[1], b[1])
    # the same 50 rows, summed by other workgroups: 50 additions each way
    assert ((a[2] - b[2]).abs() <= 2 * 66 * U * b[2]).all()


def _step(x, e, u, keep):
    s = lbm_amd.code_logits(x, e, 0.2)
    codes = lbm_amd.sample_codes(s.detach(), u, top_p=0.9)
    loss, counts, mean = lbm_amd.code_balance_loss(s, codes, keep=keep)
    total = loss + (mean * torch.log(mean + 1e-10)).sum()
    dx, de = torch.autograd.grad(total, (x, e))
    return codes, loss.detach(), counts, mean.detach(), dx, de


def _inputs(seed, N=700, D=96, K=130):
    g = gen(seed)
    return (torch.randn((N, D), generator=g).to(DEV), torch.randn((K, D), generator=g).to(DEV), torch.rand((N,), generator=g).to(DEV),
            (torch.rand((N,), generator=g) < 0.9).to(DEV))


def test_chain_equals_its_parts_and_64_bits():
    x, e, u, keep = _inputs(1)
    x.requires_grad_(), e.requires_grad_()
    codes, loss, counts, mean, dx, de = _step(x, e, u, keep)
    s = lbm_amd.code_logits(x.detach(), e.detach(), 0.2)
    want = sample64(f64(s), f64(u), np.ones(700), np.zeros(700, int), np.full(700, 0.9), np.zeros(700))
    assert np.array_equal(codes.cpu().numpy(), want)
    # the gradients by 64-bit autograd of the definition, on the codes drawn
    xr, er = x.detach().cpu().double().requires_grad_(), e.detach().cpu().double().requires_grad_()
    p = torch.softmax((2 * xr @ er.t() - (er * er).sum(1)) / 0.2, 1)[keep.cpu()].mean(0)
    f = torch.bincount(codes.cpu()[keep.cpu()], minlength=130).double()
    total = 130 * (f / f.sum() * p).sum() + (p * torch.log(p + 1e-10)).sum()
    gx, ge = torch.autograd.grad(total, (xr, er))
    # scores reach 1900 here (|x|^2 of 96 values over 0.2): they and their differences err by (96 + 8) U times that, probabilities relatively
    # as much, and the gradients are linear in those: 104 * 1900 * U = 1.2e-2 of the largest entry
    assert float((dx.cpu().double() - gx).abs().max()) <= 1.2e-2 * float(gx.abs().max())
    assert float((de.cpu().double() - ge).abs().max()) <= 1.2e-2 * float(ge.abs().max())


def test_chain_on_another_stream_and_repeated():
    x, e, u, keep = _inputs(2)
    x.requires_grad_(), e.requires_grad_()
    first = _step(x, e, u, keep)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _step(x, e, u, keep)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_two_graphs_replayed_in_turn():
    """Forward, draw and gradients captured twice, with different inputs, and replayed in turn between eager work: every replay gives the
    eager answers for what its inputs hold then."""
    graphs = []
    for seed in (3, 4):
        x, e, u, keep = _inputs(seed)
        x.requires_grad_(), e.requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(x, e, u, keep)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(x, e, u, keep)
        graphs.append((graph, x, e, u, keep, out))
    for turn in range(3):
        for graph, x, e, u, keep, out in graphs:
            with torch.no_grad():
                x.copy_(_inputs(100 + turn)[0])
                u.copy_(_inputs(200 + turn)[2])
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, _step(x, e, u, keep)):
                assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------------- in the tokenizer
def _model(shipped, **kw):
    m = lbm_amd.VQVAE(30, 256, 512, 0.25, 0.99, **kw)
    m.load_state_dict({k: torch.from_numpy(np.asarray(v)) for k, v in shipped.items()}, strict=False)
    return m.to(DEV)


@pytest.mark.parametrize("fold", [False, True])
def test_encode_with_sampling(shipped, fold):
    m = _model(shipped).eval()
    x = torch.randn((5, 30, 500), generator=gen(1)).to(DEV)
    nearest = m.encode(x, fold_projection=fold)
    B, S = nearest.shape
    # temperature 0 is the nearest code; where the two differ, the distances do by rounding only: |x|^2 + |e|^2 - 2 x.e in fp32 (256 terms)
    greedy = m.encode(x, fold_projection=fold, sampling=lbm_amd.CodeSampling(temperature=0.0), u=torch.zeros((B, S), device=DEV))
    z = lbm_amd.encoder_forward(x, m.encoder).permute(0, 2, 1).reshape(-1, 256)
    z64, e64 = f64(z), f64(m.vq_layer.embedding.weight)
    d = ((z64[:, None, :] - e64[None]) ** 2).sum(2)
    rows = np.arange(B * S)
    gap = np.abs(d[rows, greedy.cpu().numpy().ravel()] - d[rows, nearest.cpu().numpy().ravel()])
    assert (gap <= 2 * 264 * U * ((z64 ** 2).sum(1) + (e64 ** 2).sum(1).max()) * (4 if fold else 1)).all()
    # drawn codes are sample_codes of code_logits, whatever the chunking
    u = torch.rand((B, S), generator=gen(2)).to(DEV)
    hist = torch.zeros((512,), dtype=torch.int64, device=DEV)
    set_ = lbm_amd.CodeSampling(temperature=0.5, top_k=20, top_p=0.95, min_p=0.01)
    got = m.encode(x, hist=hist, fold_projection=fold, sampling=set_, u=u)
    assert got.shape == (B, S) and got.dtype == torch.int64
    assert np.array_equal(hist.cpu().numpy(), np.bincount(got.cpu().numpy().ravel(), minlength=512))
    if not fold:
        zc = lbm_amd.encoder_forward(x, m.encoder, pitched_out=True)
        scores = lbm_amd.code_logits(zc, m.vq_layer.embedding.weight.detach(), channel_major=True)
        want = lbm_amd.sample_codes(scores, u.reshape(-1), temperature=0.5, top_k=20, top_p=0.95, min_p=0.01)
        assert torch.equal(got.reshape(-1), want)
        assert np.array_equal(want.cpu().numpy(), sample64(f64(scores), f64(u).ravel(), np.full(B * S, 0.5), np.full(B * S, 20), np.full(B * S, 0.95),
                                                           np.full(B * S, 0.01)))
    # codes that may not be drawn are not; numbers from a generator repeat with its seed
    allowed = torch.zeros((512,), dtype=torch.bool, device=DEV)
    allowed[[3, 77, 200]] = True
    only = lbm_amd.CodeSampling(temperature=10.0, allowed=allowed)
    a = m.encode(x, fold_projection=fold, sampling=only, generator=torch.Generator(device=DEV).manual_seed(5))
    b = m.encode(x, fold_projection=fold, sampling=only, generator=torch.Generator(device=DEV).manual_seed(5))
    assert torch.equal(a, b) and set(a.unique().tolist()) <= {3, 77, 200}
    for kw in (dict(screened=True, sampling=set_), dict(u=u), dict(sampling=set_, u=u[:, :-1])):
        with pytest.raises(ValueError):
            m.encode(x, fold_projection=fold, **kw)


def test_encode_with_settings_per_position_in_runs_of_epochs(shipped, monkeypatch):
    import lbm_amd.quantizer as quantizer
    m = _model(shipped).eval()
    x = torch.randn((5, 30, 200), generator=gen(11)).to(DEV)
    B, S = m.encode(x).shape
    g = gen(12)
    set_ = lbm_amd.CodeSampling(temperature=(torch.rand((B, S), generator=g) + 0.2).to(DEV), top_k=torch.randint(0, 40, (B, S), generator=g).to(DEV),
                                top_p=(0.5 + 0.5 * torch.rand((B, S), generator=g)).to(DEV), min_p=(0.05 * torch.rand((B, S), generator=g)).to(DEV),
                                allowed=(torch.rand((B, S, 512), generator=g) < 0.8).to(DEV))
    u = torch.rand((B, S), generator=g).to(DEV)
    whole = m.encode(x, sampling=set_, u=u)
    monkeypatch.setattr(quantizer, "_SCORES_AT_A_TIME", 2 * S * 512)
    assert torch.equal(m.encode(x, sampling=set_, u=u), whole)
    assert set_.allowed.gather(2, whole[..., None]).all()
    with pytest.raises(ValueError):
        m.encode(x[:4], sampling=set_, u=u[:4])


def test_encode_data_for_transformer_with_sampling(shipped):
    m = _model(shipped)
    data = [(torch.randn((2, 30, 100), generator=gen(i)), torch.tensor([i, i])) for i in range(3)]
    one = lbm_amd.encode_data_for_transformer(m, data, DEV, sampling=lbm_amd.CodeSampling(temperature=2.0),
                                              generator=torch.Generator(device=DEV).manual_seed(1))
    two = lbm_amd.encode_data_for_transformer(m, data, DEV, sampling=lbm_amd.CodeSampling(temperature=2.0),
                                              generator=torch.Generator(device=DEV).manual_seed(1))
    assert one[0].shape == (6, 25) and one[0].dtype == np.int64 and np.array_equal(one[0], two[0]) and one[1].tolist() == [0, 0, 1, 1, 2, 2]
    assert not np.array_equal(one[0], lbm_amd.encode_data_for_transformer(m, data, DEV)[0])


def test_quantizer_training_step_with_balance():
    """The balance term's gradient reaches the inputs through the codebook as it was BEFORE the step's EMA update, which itself is the one
    without the term."""
    N, D, K, wgt, T = 96, 16, 24, 0.7, 0.5
    x = torch.randn((4, N // 4, D), generator=gen(1))
    results = {}
    for weight in (0.0, wgt):
        torch.manual_seed(3)
        q = lbm_amd.VectorQuantizerEMA(K, D, 0.25, 0.9, balance_weight=weight, balance_temperature=T)
        q.embedding.weight.data.normal_(generator=gen(2))
        q.ema_w.data.copy_(q.embedding.weight.data)
        q.ema_cluster_size.data.fill_(1.0)
        before = q.embedding.weight.detach().clone().double()
        q = q.to(DEV).train()
        xd = x.to(DEV).requires_grad_()
        loss, _, _, idx = q(xd)
        loss.backward()
        results[weight] = (loss.detach(), xd.grad, idx, q.embedding.weight.detach().clone(), q.ema_w.clone())
    l0, g0, i0, w0, m0 = results[0.0]
    l1, g1, i1, w1, m1 = results[wgt]
    assert torch.equal(i0, i1) and torch.equal(w0, w1) and torch.equal(m0, m1)
    assert not torch.equal(w1.cpu().double(), before)
    xr = x.double().reshape(N, D).requires_grad_()
    p = torch.softmax((2 * xr @ before.t() - (before * before).sum(1)) / T, 1).mean(0)
    f = torch.bincount(i1.cpu().reshape(-1), minlength=K).double() / N
    term = wgt * K * (f * p).sum()
    (want,) = torch.autograd.grad(term, xr)
    # scores up to some 100 err by 24 U of that, probabilities and gradients relatively as much: 2e-4; the differences of two fp32 results
    assert abs(float(l1 - l0) - float(term.detach())) <= 2e-4 * float(term.detach()) + 4 * U * abs(float(l1))
    err = (g1 - g0).cpu().double().reshape(N, D) - want
    assert float(err.abs().max()) <= 2e-4 * float(want.abs().max()) + 4 * U * float(g1.abs().max())
    # not in eval mode
    q.eval()
    with torch.no_grad():
        a = q(x.to(DEV))[0]
        q.balance_weight = 0.0
        assert torch.equal(a, q(x.to(DEV))[0])
