"""The code-score operators on the GPU where scores, operands and sizes go to their ends: best codes far above a row's other scores, operands
near the largest float, more rows or gradient entries than one launch holds.  Plain 64-bit evaluations and tolerances as in test_gpu_codes."""
import contextlib

import numpy as np
import pytest
import torch

import lbm_amd
from tests.test_gpu_codes import DEV, TYPES, U, f64, gen, logits64, logits_tol, sample64

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
