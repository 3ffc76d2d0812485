"""The code-score operators on the GPU where scores, operands and sizes go to their ends: best codes far above a row's other scores, operands
near the largest float, more rows or gradient entries than one launch holds.  Plain 64-bit evaluations and tolerances as in test_gpu_codes."""
import contextlib

import numpy as np
import pytest
import torch

import lbm_amd
from tests.test_gpu_codes import DEV, TYPES, U, _inputs, _step, f64, gen, logits64, logits_tol, sample64

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("T", [1.0, 0.25])
@pytest.mark.parametrize("K", [1500, 8192, 8191])
def test_sample_nucleus_of_best_codes_far_above_the_rest(K, T, kind):
    """Two to four best codes, equal or nearly so, 80 to 95 T above every other score and off the columns i K / 512 that are looked at first."""
    g = gen(K)
    looked_at = torch.arange(512) * K // 512
    off = torch.ones((K,), dtype=torch.bool)
    off[looked_at] = False
    off = off.nonzero()[:, 0]
    gaps = torch.cat([torch.arange(80.0, 96.0), torch.arange(86.5, 89.5, 0.125)])
    n = gaps.numel()
    for best in (2, 3, 4):
        s = -torch.rand((n, K), generator=g) * T               # at most 0
        s[:, looked_at[100]] = 0.0                             # the best of the columns looked at
        at = off[torch.stack([torch.randperm(off.numel(), generator=g)[:best] for _ in range(n)])]
        step = 0.25 * T * torch.randint(0, 2, (n, best), generator=g)
        s.scatter_(1, at, (gaps * T)[:, None] + step)
        st = s.to(TYPES[kind])
        for u in (0.0, 0.3, 0.5, 0.7, 0.999):
            for p in (0.9, 0.55):
                ut = torch.full((n,), u)
                got = lbm_amd.sample_codes(st.to(DEV), ut.to(DEV), temperature=T, top_p=p).cpu().numpy()
                assert (got[:, None] == at.numpy()).any(1).all()
                # u = 1/2 meets a border exactly where the weights on its two sides are the same ones (1 + w and 1 + w, say), and either side
                # may then be answered: a weight errs by 4 2^-53 of itself at most (its exponent's product, the polynomial, the last
                # rounding; exponents here are at most 1), the sums of up to four of them and the product with u by 4 2^-53 of the total
                # more, on each of the two evaluations: 16 2^-53 of the total in all.  u moved by that much to either side brackets it.
                lo, hi = (sample64(f64(st), f64(ut) + d, np.full(n, T), np.zeros(n, int), np.full(n, p), np.zeros(n)) for d in (-2.0 ** -49, 2.0 ** -49))
                assert ((got == lo) | (got == hi)).all(), (best, u, p, got, lo, hi)


def test_sample_numbers_in_64_bits_stay_below_one():
    """Numbers of [0, 1) that round to 1 in fp32 are the last fp32 number below it: the code that a share of 1 - 2^-24 falls on, not a code
    without weight to speak of behind it."""
    for K in (2, 700, 5000):
        s = torch.full((4, K), float("-inf"))
        s[:, 0], s[:, K - 1] = 0.0, -100.0
        u = torch.tensor([1 - 1e-9, 1 - 2.0 ** -53, 0.25, 1.0], dtype=torch.float64)
        for kw in (dict(), dict(top_k=2), dict(top_p=0.999999999999)):
            got = lbm_amd.sample_codes(s.to(DEV), u.to(DEV), **kw).tolist()
            assert got[:3] == [0, 0, 0]
        assert lbm_amd.sample_codes(s.to(DEV), u.to(DEV)).tolist()[3] == K - 1       # 1 itself: the last code that stayed


# ------------------------------------------------------------------------------------------------------------- gradients
@pytest.mark.parametrize("kind", sorted(TYPES))
def test_gradients_with_saved_tensors_offloaded(kind):
    """Saved tensors that went to host memory come back dense: gradients are those without, bit for bit, whatever the scores' row stride was."""
    g = gen(31)
    wide = torch.randn((90, 700), generator=g).to(TYPES[kind]).to(DEV)
    codes = torch.randint(0, 130, (90,), generator=g).to(DEV)
    e = torch.randn((70, 130), generator=g).to(DEV).requires_grad_()
    gm, gs = torch.randn((130,), generator=g).to(DEV), torch.randn((90, 70), generator=g).to(DEV)
    for at in (0, 3):
        results = []
        for offload in (False, True):
            s = wide[:, at:at + 130].detach().requires_grad_()
            with torch.autograd.graph.save_on_cpu() if offload else contextlib.nullcontext():
                loss, _, mean = lbm_amd.code_balance_loss(s, codes)
                out = lbm_amd.code_logits(s.float(), e, 0.5)
            results.append(torch.autograd.grad((loss, mean), s, (torch.ones((), device=DEV), gm)) + torch.autograd.grad(out, (s, e), gs))
        for a, b in zip(*results):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------------- scores
@pytest.mark.parametrize("D,K,N", [(1, 3, 5), (64, 96, 70), (65, 97, 130), (256, 512, 1000)])
def test_logits_of_operands_near_the_largest_float(D, K, N):
    """Operands up to the last float that rounds to a finite bf16 number give what the formula gives; the next one, the largest float and an
    infinity give NaN in their own row or column and nowhere else."""
    last = float(np.uint32(0x7f7f7fff).view(np.float32))
    g = gen(D)
    x, e = torch.randn((N, D), generator=g) * 1e-3, torch.randn((K, D), generator=g) * 1e-3
    x[::3, D // 2], x[1::3, 0] = last, -last
    w = torch.randn((N, K), generator=g) * 1e-3
    w[N // 2, K // 2] = -last
    xd, ed = x.to(DEV).requires_grad_(), e.to(DEV).requires_grad_()
    s = lbm_amd.code_logits(xd, ed, 0.5)
    x64, e64, w64 = f64(x), f64(e), f64(w)
    assert (np.abs(f64(s) - logits64(x64, e64, 0.5)) <= logits_tol(x64, e64, 0.5)).all()
    (dx,) = torch.autograd.grad(s, xd, w.to(DEV))
    assert (np.abs(f64(dx) - 4 * w64 @ e64) <= U * (K + 8) * 4 * (np.abs(w64) @ np.abs(e64)) + 1e-37).all()
    for value in (float(np.uint32(0x7f7f8000).view(np.float32)), -torch.finfo(torch.float32).max, float("inf")):
        for channel_major in (False, True):
            a, b = x.clone(), e.clone()
            a[N - 2, D - 1], b[K - 2, 0] = value, value
            a = (a.t()[None] if channel_major else a).contiguous()
            t = lbm_amd.code_logits(a.to(DEV), b.to(DEV), 0.5, channel_major=channel_major).cpu()
            other = torch.ones((N, K), dtype=torch.bool)
            other[N - 2] = other[:, K - 2] = False
            assert torch.isnan(t[~other]).all()
            assert (np.abs(f64(t) - logits64(x64, e64, 0.5))[other] <= logits_tol(x64, e64, 0.5)[other]).all()
        v = torch.randn((N, K), generator=g)
        v[N - 2, K - 1] = value
        y = x.clamp(-1, 1)
        yd = y.to(DEV).requires_grad_()
        dx, de = (t.cpu() for t in torch.autograd.grad(lbm_amd.code_logits(yd, ed, 0.5), (yd, ed), v.to(DEV)))
        assert torch.isnan(dx[N - 2]).all() and torch.isfinite(dx[torch.arange(N) != N - 2]).all()
        assert torch.isnan(de[K - 1]).all() and torch.isfinite(de[:K - 1]).all()


# ---------------------------------------------------------------------------------------------------------- large extents
def test_sample_more_rows_than_one_launch_holds():
    """Row counts whose waves are more than 2^32 threads: every row is answered, with its own settings, mask and number."""
    if torch.cuda.get_device_properties(0).total_memory < 20e9:
        pytest.skip("needs 8 GB of device memory")
    N = (1 << 26) + 1001
    g = torch.Generator(device=DEV).manual_seed(1)
    s = torch.randn((N, 3), generator=g, device=DEV, dtype=torch.bfloat16)
    u = torch.rand((N,), generator=g, device=DEV)
    allowed = torch.rand((N, 3), generator=g, device=DEV) < 0.7
    k = torch.randint(0, 3, (N,), generator=g, device=DEV, dtype=torch.int32)
    hist = torch.zeros((3,), dtype=torch.int64, device=DEV)
    got = lbm_amd.sample_codes(s, u, top_k=k, allowed=allowed, hist=hist)
    for a in (0, 1 << 25, N // 2, (1 << 26) - 5, N - 1001):
        b = slice(a, a + 1001)
        assert torch.equal(got[b], lbm_amd.sample_codes(s[b], u[b], top_k=k[b], allowed=allowed[b]))
    assert torch.equal(hist, torch.stack([(got == i).sum() for i in range(3)]))


def test_logits_gradients_of_more_entries_than_one_launch_holds():
    """Gradients of more than 2^32 entries that are joined from pieces."""
    if torch.cuda.get_device_properties(0).total_memory < 120e9:
        pytest.skip("needs 70 GB of device memory")
    D, n, m = 8192, (1 << 19) + 1000, 3
    g = torch.Generator(device=DEV).manual_seed(1)
    big = torch.empty((n, D), device=DEV).normal_(generator=g)
    w = torch.randn((m, n), generator=g, device=DEV)
    small = torch.randn((m, D), generator=g, device=DEV)

    def close(got, rows, want, mag, steps):
        assert ((got[rows].double() - want).abs() <= U * (steps + 16) * mag + 1e-37).all()
    rows = torch.tensor([0, 1, 77, (1 << 19) - 1, 1 << 19, n - 2, n - 1], device=DEV)
    # the codebook's gradient
    e = big.requires_grad_()
    (de,) = torch.autograd.grad(lbm_amd.code_logits(small, e, 1.0), e, w)
    wr = w[:, rows].double().t().contiguous()
    er, c = big.detach()[rows].double(), wr.sum(1)[:, None]
    close(de, rows, 2 * (torch.mm(wr, small.double()) - c * er), 2 * (torch.mm(wr.abs(), small.double().abs()) + wr.abs().sum(1)[:, None] * er.abs()), m)

    # the rows' gradient: the codes in more than one piece
    del de, e
    x, cb = big.detach().requires_grad_(), torch.randn((4100, D), generator=g, device=DEV)
    w = torch.zeros((n, 4100), device=DEV)
    w[rows] = torch.randn((7, 4100), generator=g, device=DEV)
    (dx,) = torch.autograd.grad(lbm_amd.code_logits(x, cb, 1.0), x, w)
    wr = w[rows].double()
    close(dx, rows, 2 * torch.mm(wr, cb.double()), 2 * torch.mm(wr.abs(), cb.double().abs()), 4100)
    assert not dx[2:70].any() and not dx[-90:-3].any()


# ------------------------------------------------------------------------------------------------------ together, in training
def test_chain_gradients_of_scores_of_ordinary_size():
    """Scores -> drawn codes -> loss and entropy of the mean -> gradients, every entry within a bound from the operations: scores of a few units,
    so that every code has a share of every row."""
    T, N, D, K = 0.2, 700, 96, 130                      # those of _step and _inputs
    x, e, u, keep = _inputs(5)
    x, e = (x * 0.15).requires_grad_(), (e * 0.15).requires_grad_()
    codes, loss, counts, mean, dx, de = _step(x, e, u, keep)
    x64, e64, on = f64(x), f64(e), keep.cpu().numpy()
    s = logits64(x64, e64, T)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    assert np.median(p.max(1)) < 0.5
    M = on.sum()
    f = np.bincount(codes.cpu().numpy()[on], minlength=K)
    assert np.array_equal(counts.cpu().numpy(), f)
    f = f / f.sum()
    P = p[on].mean(0)
    a = K * f + np.log(P + 1e-10) + P / (P + 1e-10)
    ds = np.where(on[:, None], p * (a - (p * a).sum(1, keepdims=True)) / M, 0)
    # relative error of a row's p: its scores' errors twice (its own and the sum's), then the exponential, the sum of 130 and the reciprocal;
    # of P: the worst row's and the sum over the rows; of a: that of P in the logarithm (absolutely) and in P / P, and the roundings of its parts
    r = 2 * logits_tol(x64, e64, T).max(1) + 64 * U
    rP = r[on].max() + (N + 16) * U
    ta = 3 * rP + 8 * U * (K * f + np.abs(np.log(P + 1e-10)) + 1)
    assert (np.abs(f64(mean) - P) <= rP * P).all()
    assert abs(float(loss) - K * (f * P).sum()) <= (rP + 4 * U) * K * (f * P).sum()
    dev = np.abs(a - (p * a).sum(1, keepdims=True))
    inner = (p * (r[:, None] * dev + ta)).sum(1, keepdims=True)      # of p.a (p's errors sum to nothing but rounding: a is taken from its mean)
    tds = np.where(on[:, None], p * (r[:, None] * dev + ta + inner + 64 * U * np.abs(a).max()) / M, 0)
    gx, ge = 2 / T * ds @ e64, 2 / T * (ds.T @ x64 - ds.sum(0)[:, None] * e64)
    tx = 2 / T * (tds @ np.abs(e64) + U * (K + 8) * np.abs(ds) @ np.abs(e64))
    mag = np.abs(ds).T @ np.abs(x64) + np.abs(ds).sum(0)[:, None] * np.abs(e64)
    te = 2 / T * (tds.T @ np.abs(x64) + tds.sum(0)[:, None] * np.abs(e64) + U * (N + 16) * mag)
    assert (np.abs(f64(dx) - gx) <= tx).all() and (np.abs(f64(de) - ge) <= te).all()
    # what the bounds can tell apart: a twentieth of an ordinary entry
    assert np.median(tx[on] / np.abs(gx[on]).clip(1e-30)) < 0.05 and np.median(te / np.abs(ge).clip(1e-30)) < 0.05


def test_balance_term_takes_this_ranks_rows_where_the_ema_step_is_summed_over_ranks(monkeypatch):
    x = torch.randn((96, 16), generator=gen(1)).to(DEV)
    results = []
    for group in (None, "all"):
        if group is not None:
            monkeypatch.setattr(torch.distributed, "all_reduce", lambda t, group=None: t.mul_(3))     # two more ranks with the same rows
        q = lbm_amd.VectorQuantizerEMA(24, 16, 0.25, 0.9, balance_weight=0.7, balance_temperature=0.5)
        q.embedding.weight.data.normal_(generator=gen(2))
        q.ema_w.data.copy_(q.embedding.weight.data)
        q.ema_cluster_size.data.fill_(1.0)
        q.ema_group = group
        q = q.to(DEV).train()
        xd = x.clone().requires_grad_()
        loss, _, _, _ = q(xd)
        loss.backward()
        results.append((loss.detach(), xd.grad, q.embedding.weight.detach().clone()))
    (l0, g0, w0), (l1, g1, w1) = results
    assert torch.equal(l0, l1) and torch.equal(g0, g1) and not torch.equal(w0, w1)


@pytest.mark.parametrize("B,S,K", [(5, 5, 3), (7, 130, 70), (300, 1, 33), (1, 9, 4)])
def test_logits_channel_major_of_one_channel(B, S, K):
    """One channel: the stride of that dimension is any number, here that of the whole tensor, of one element, of a wider row."""
    g = gen(B)
    z, e = torch.randn((B, 1, S), generator=g), torch.randn((K, 1), generator=g)
    d = z.to(DEV)
    wide = torch.zeros((B, 3, S + 5), device=DEV)
    wide[:, 1:2, 2:2 + S] = d
    want, tol = logits64(f64(z).reshape(-1, 1), f64(e), 0.5), logits_tol(f64(z).reshape(-1, 1), f64(e), 0.5)
    for x in (d, d.view(1, B, S).transpose(0, 1), d.view(B, S, 1).permute(0, 2, 1), wide[:, 1:2, 2:2 + S], wide[:, 1:2, 2:2 + S].transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(x, d)
        assert (np.abs(f64(lbm_amd.code_logits(x, e.to(DEV), 0.5, channel_major=True)) - want) <= tol).all()
