"""Refusals of the code-score operators (code_logits, code_balance_loss, sample_codes) and of their C entry points: no GPU, no launch."""
import math

import pytest
import torch

import lbm_amd
from lbm_amd import _lib

EINVAL, EUNSUPPORTED = -1, -2
P = 4096      # stands for a device pointer in calls that are refused before it is used


def _err():
    return _lib.load().lbm_last_error().decode()


def _logits(x=P, ldx=8, layout=0, S=0, cb=P, ee=None, out=P, ldl=16, N=4, D=8, K=16, T=1.0):
    return _lib.load().lbm_code_logits_f32(x, ldx, layout, S, cb, ee, out, ldl, N, D, K, T, None)


@pytest.mark.parametrize("kw", [dict(N=-1), dict(D=0), dict(K=0), dict(T=0.0), dict(T=-1.0), dict(T=math.inf), dict(T=math.nan), dict(layout=2),
                                dict(layout=-1), dict(x=None), dict(cb=None), dict(out=None), dict(ldl=15), dict(ldx=7),
                                dict(layout=1, S=0), dict(layout=1, S=3), dict(layout=1, S=4, ldx=3)])
def test_logits_entry_refuses(kw):
    assert _logits(**kw) == EINVAL and "lbm_code_logits_f32" in _err()


def test_logits_entry_empty():
    assert _logits(N=0, x=None, out=None) == 0


def _grad(g=P, ldg=16, x=P, ldx=8, cb=P, dx=P, de=P, norm=1, ws=P, N=4, D=8, K=16, T=1.0):
    return _lib.load().lbm_code_logits_grad_f32(g, ldg, x, ldx, cb, dx, de, norm, ws, N, D, K, T, None)


@pytest.mark.parametrize("kw", [dict(N=-1), dict(D=0), dict(K=0), dict(T=0.0), dict(T=math.nan), dict(g=None), dict(cb=None), dict(ldg=15),
                                dict(x=None), dict(ws=None), dict(ldx=7), dict(ws=P + 8), dict(de=None, ws=None)])
def test_logits_grad_entry_refuses(kw):
    assert _grad(**kw) == EINVAL and "lbm_code_logits_grad_f32" in _err()


def test_logits_grad_entry_without_outputs():
    assert _grad(dx=None, de=None, x=None, ws=None) == 0
    assert _lib.load().lbm_code_logits_grad_workspace_bytes(-1, 8, 16) == 0
    assert _lib.load().lbm_code_logits_grad_workspace_bytes(0, 8, 16) > 0


def _balance(s=P, dt=0, lds=16, codes=P, slots=1, keep=None, loss=P, counts=P, mean=P, stat=P, tot=P, ws=P, N=4, K=16):
    return _lib.load().lbm_code_balance(s, dt, lds, codes, slots, keep, loss, counts, mean, stat, tot, ws, N, K, None)


@pytest.mark.parametrize("kw,rc", [(dict(N=-1), EINVAL), (dict(K=0), EINVAL), (dict(K=8193), EUNSUPPORTED), (dict(dt=3), EINVAL),
                                   (dict(dt=-1), EINVAL), (dict(s=None), EINVAL), (dict(loss=None), EINVAL), (dict(counts=None), EINVAL),
                                   (dict(mean=None), EINVAL), (dict(stat=None), EINVAL), (dict(stat=P + 4), EINVAL), (dict(tot=None), EINVAL),
                                   (dict(ws=None), EINVAL), (dict(ws=P + 8), EINVAL), (dict(lds=-16), EINVAL), (dict(slots=0), EINVAL)])
def test_balance_entry_refuses(kw, rc):
    assert _balance(**kw) == rc and "lbm_code_balance" in _err()


def _balance_grad(s=P, dt=0, lds=16, stat=P, counts=P, tot=P, gl=P, gm=P, ds=P, N=4, K=16):
    return _lib.load().lbm_code_balance_grad(s, dt, lds, stat, counts, tot, gl, gm, ds, N, K, None)


@pytest.mark.parametrize("kw,rc", [(dict(N=-1), EINVAL), (dict(K=0), EINVAL), (dict(K=8193), EUNSUPPORTED), (dict(dt=7), EINVAL),
                                   (dict(s=None), EINVAL), (dict(stat=None), EINVAL), (dict(counts=None), EINVAL), (dict(tot=None), EINVAL),
                                   (dict(ds=None), EINVAL), (dict(lds=-1), EINVAL)])
def test_balance_grad_entry_refuses(kw, rc):
    assert _balance_grad(**kw) == rc and "lbm_code_balance_grad" in _err()


def test_balance_grad_entry_empty():
    assert _balance_grad(N=0, s=None, stat=None, ds=None) == 0
    lib = _lib.load()
    assert lib.lbm_code_balance_workspace_bytes(1, 8193) == 0 and lib.lbm_code_balance_workspace_bytes(-1, 8) == 0
    assert lib.lbm_code_balance_workspace_bytes(0, 8) > 0


def _sample(s=P, dt=0, lds=16, u=P, tr=None, t=1.0, kr=None, k=0, pr=None, p=1.0, mr=None, m=0.0, al=None, ald=0, out=P, hist=None, N=4, K=16):
    return _lib.load().lbm_code_sample(s, dt, lds, u, tr, t, kr, k, pr, p, mr, m, al, ald, out, hist, N, K, None)


@pytest.mark.parametrize("kw,rc", [(dict(N=-1), EINVAL), (dict(K=0), EINVAL), (dict(K=(1 << 24) + 1), EUNSUPPORTED),
                                   (dict(K=32769, hist=P), EUNSUPPORTED), (dict(dt=3), EINVAL), (dict(t=-0.5), EINVAL), (dict(t=math.nan), EINVAL), (dict(k=-1), EINVAL), (dict(p=-0.1), EINVAL),
                                   (dict(p=1.1), EINVAL), (dict(p=math.nan), EINVAL), (dict(m=-0.1), EINVAL), (dict(m=1.5), EINVAL),
                                   (dict(s=None), EINVAL), (dict(u=None), EINVAL), (dict(out=None), EINVAL), (dict(lds=-16), EINVAL),
                                   (dict(al=P, ald=-16), EINVAL), (dict(N=1 << 31), EUNSUPPORTED)])
def test_sample_entry_refuses(kw, rc):
    assert _sample(**kw) == rc and "lbm_code_sample" in _err()


def test_sample_entry_empty():
    assert _sample(N=0, s=None, u=None, out=None) == 0


# ---- the Python surface: every refusal comes before a tensor is touched, so CPU tensors do
S = torch.zeros((4, 16))
U = torch.zeros((4,))


@pytest.mark.parametrize("call", [
    lambda: lbm_amd.sample_codes(S, torch.zeros((5,))),
    lambda: lbm_amd.sample_codes(S, torch.zeros((4,), dtype=torch.int64)),
    lambda: lbm_amd.sample_codes(S.double(), U),
    lambda: lbm_amd.sample_codes(torch.zeros((4, 0)), U),
    lambda: lbm_amd.sample_codes(S, U, temperature=-1.0),
    lambda: lbm_amd.sample_codes(S, U, temperature=math.nan),
    lambda: lbm_amd.sample_codes(S, U, temperature=torch.ones((3,))),
    lambda: lbm_amd.sample_codes(S, U, top_k=-1),
    lambda: lbm_amd.sample_codes(S, U, top_k=2.5),
    lambda: lbm_amd.sample_codes(S, U, top_k=torch.ones((4,))),
    lambda: lbm_amd.sample_codes(S, U, top_p=1.5),
    lambda: lbm_amd.sample_codes(S, U, min_p=-0.1),
    lambda: lbm_amd.sample_codes(S, U, allowed=torch.ones((15,), dtype=torch.bool)),
    lambda: lbm_amd.sample_codes(S, U, allowed=torch.ones((16,))),
    lambda: lbm_amd.sample_codes(S, U, hist=torch.zeros((16,))),
    lambda: lbm_amd.code_balance_loss(S.double()),
    lambda: lbm_amd.code_balance_loss([1.0, 2.0]),
    lambda: lbm_amd.code_balance_loss(S, torch.zeros((4,))),
    lambda: lbm_amd.code_balance_loss(S, torch.zeros((3,), dtype=torch.int64)),
    lambda: lbm_amd.code_balance_loss(S, torch.zeros((4, 0), dtype=torch.int64)),
    lambda: lbm_amd.code_balance_loss(S, keep=torch.ones((4,))),
    lambda: lbm_amd.code_balance_loss(S, keep=torch.ones((3,), dtype=torch.bool)),
    lambda: lbm_amd.code_logits(S, S, temperature=0.0),
    lambda: lbm_amd.code_logits(S, S, temperature=math.inf),
])
def test_python_surface_refuses(call):
    with pytest.raises(ValueError):
        call()


def test_python_surface_refuses_cpu_tensors():
    for call in (lambda: lbm_amd.sample_codes(S, U), lambda: lbm_amd.code_balance_loss(S)):
        with pytest.raises(_lib.LbmError, match="CUDA/ROCm"):
            call()
    with pytest.raises(NotImplementedError, match="8192"):
        lbm_amd.code_balance_loss(torch.zeros((1, 8193)))


class _Recorder:
    """Stands for the library: every call succeeds and is written down, nothing is touched."""
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 64 if name.endswith("_bytes") else 0
        return call


@pytest.mark.parametrize("op", ["balance", "logits"])
@pytest.mark.parametrize("wide", [False, True])
def test_backward_addresses_saved_tensors_as_they_come_back(monkeypatch, op, wide):
    """Saved tensors may come back in another layout than they went (offloading to host memory makes them dense, a hook may also spread
    them): the backward pass goes by the strides they have then."""
    rec = _Recorder()
    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(_lib, "ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(_lib, "stream_ptr", lambda: 0)
    monkeypatch.setattr(_lib, "dev_f32", lambda t, device=None: t.float().contiguous())
    N, K, D = 6, 16, 16
    back = []

    def unpack(t):
        if t.dtype == torch.float32 and t.dim() == 2:
            t = torch.zeros((t.shape[0], 4 * t.shape[1]))[:, ::4] if wide else t.clone(memory_format=torch.contiguous_format)
        back.append(t)
        return t
    x = torch.zeros((N, 100))[:, 3:3 + K].requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        if op == "balance":
            out = lbm_amd.code_balance_loss(x)[0]
        else:
            out = lbm_amd.code_logits(x, torch.zeros((K, D)).requires_grad_()).sum()
    out.backward()
    name, args = rec.calls[-1]
    stride, pointers = (args[2], args[:1]) if op == "balance" else (args[3], (args[2], args[4]))
    assert name == ("lbm_code_balance_grad" if op == "balance" else "lbm_code_logits_grad_f32")
    assert stride == K
    if not wide:
        assert set(pointers) <= {t.data_ptr() for t in back}
    else:
        assert not set(pointers) & {t.data_ptr() for t in back}      # dense copies of rows whose scores are not neighbours


@pytest.mark.parametrize("T", [1e-300, 5e-324, 1e-39, 2.0 / torch.finfo(torch.float32).max * (1 - 1e-12)])
def test_temperatures_whose_reciprocal_is_no_float_are_refused(T):
    assert _logits(T=T) == EINVAL and "2 / temperature" in _err()
    assert _grad(T=T) == EINVAL and "2 / temperature" in _err()
    with pytest.raises(ValueError, match="2 / temperature"):
        lbm_amd.code_logits(S, S, temperature=T)


def test_smallest_temperatures_are_taken():
    assert _logits(T=6e-39, N=0) == 0 and _grad(T=6e-39, dx=None, de=None, x=None, ws=None) == 0


def test_balance_grad_entry_refuses_unaligned_row_statistics():
    assert _balance_grad(stat=P + 4) == EINVAL and "lbm_code_balance_grad: row_stat" in _err()


def test_pitch_of_a_single_channel_is_the_distance_of_the_epochs():
    """[B, 1, L] views whose middle stride, of a dimension of one, is any number: the pitch the kernels are given stays inside the tensor."""
    from lbm_amd.quantizer import _pitched_rows
    base = torch.arange(1000.0)
    for B, L in ((5, 7), (2, 1), (1, 6), (5, 8)):
        for s0 in (L, L + 1, 8, 1, 0):
            for s1 in (0, 1, L, B * L, 900):
                x = torch.as_strided(base, (B, 1, L), (s0, s1, 1))
                y = _pitched_rows(x)
                assert torch.equal(x, y)
                if B > 1:      # what conv1d, vq_argmin and code_logits hand over as the pitch
                    assert y.stride(1) == y.stride(0) >= L and (L == 1 or y.stride(2) == 1)
    y = _pitched_rows(base[:35].view(1, 5, 7).transpose(0, 1))
    assert y.stride(1) == 7 and y.data_ptr() == base.data_ptr()
