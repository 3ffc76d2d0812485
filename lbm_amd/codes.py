"""Scores of the codebook's codes and what is made of them: the scores as a matrix with gradients, a usage-balance loss, and codes drawn
from the scores.

The reference decides every code by argmin (training/model.py:90-95, 152-158) and only measures collapse (perplexity, :142-144); its
shipped codebook has 100 codes of 512 that are never used.  ``code_logits`` + ``code_balance_loss`` give training a term that works
against it (``VectorQuantizerEMA(balance_weight=...)``); ``code_logits`` + ``sample_codes`` tokenize by a draw instead of the argmin
(``VQVAE.encode(sampling=...)``), and ``sample_codes`` alone draws the next code from any model's scores over codes.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _lib

_F32_MAX = torch.finfo(torch.float32).max


# --------------------------------------------------------------------------------------------------------------- scores
def _rows(t: torch.Tensor):
    """[N, M] as (tensor with unit stride along M, row stride of M at least)."""
    (n, m), (ld, unit) = t.shape, t.stride()
    if unit != 1 or (n > 1 and ld < m):
        t, ld = t.contiguous(), m
    return t, (ld if n > 1 else m)


class _CodeLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ldx, codebook, e_sqnorm, temperature):
        N, D = x.shape
        K = codebook.shape[0]
        out = torch.empty((N, K), dtype=torch.float32, device=x.device)
        _lib.check(_lib.load().lbm_code_logits_f32(_lib.ptr(x), ldx, _lib.VQ_ROWS, 0, _lib.ptr(codebook), _lib.ptr(e_sqnorm),
                                                   out.data_ptr(), K, N, D, K, temperature, _lib.stream_ptr()),
                   "lbm_code_logits_f32")
        ctx.save_for_backward(x, codebook)
        ctx.temperature, ctx.norm_grad = temperature, e_sqnorm is None
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, codebook = ctx.saved_tensors
        need_x, _, need_e = ctx.needs_input_grad[:3]
        N, D = x.shape
        K = codebook.shape[0]
        # saved tensors come back in any layout from hooks that offload them
        (g, ldg), (x, ldx), codebook = _rows(g), _rows(x), codebook.contiguous()
        if not g.get_device() == x.get_device() == codebook.get_device():
            raise _lib.LbmError("code_logits: saved tensors came back on another device")
        lib = _lib.load()
        dx = torch.empty((N, D), dtype=torch.float32, device=x.device) if need_x else None
        de = torch.empty((K, D), dtype=torch.float32, device=x.device) if need_e else None
        ws = torch.empty((lib.lbm_code_logits_grad_workspace_bytes(N, D, K),), dtype=torch.uint8, device=x.device)
        _lib.check(lib.lbm_code_logits_grad_f32(_lib.ptr(g), ldg, x.data_ptr(), ldx, codebook.data_ptr(), dx.data_ptr() if need_x else None,
                                                de.data_ptr() if need_e else None, int(ctx.norm_grad), ws.data_ptr(), N, D, K,
                                                ctx.temperature, _lib.stream_ptr()), "lbm_code_logits_grad_f32")
        return dx, None, de, None, None


def _f32_param(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        return _lib.dev_f32(t)
    if not t.is_floating_point():
        raise ValueError(f"{what} must be a floating-point tensor")
    return t if t.dtype is torch.float32 else t.to(torch.float32)


@_lib.on_tensor_device
def code_logits(x: torch.Tensor, codebook: torch.Tensor, temperature: float = 1.0, *, e_sqnorm: torch.Tensor = None,
                channel_major: bool = False) -> torch.Tensor:
    """Scores of all codes: ``out[n, k] = (2 x_n.e_k - |e_k|^2) / temperature``, float32 [N, K].

    That is minus the squared distance over ``temperature`` up to a constant of the row, so softmax, argmax and every ranking of a row are
    those of the distances.  ``x``: [N, D] rows (any row stride), or with ``channel_major`` the encoder output z[B, D, S] (N = B*S rows, row
    n = (n // S, n % S), no permute copy).  Differentiable in ``x`` and ``codebook``; with ``channel_major`` and a gradient to take, the
    rows are copied first.  ``e_sqnorm`` ([K], as ``fold_projection`` returns it) takes the place of |e_k|^2 as a constant.
    Values of 3.396e38 and more in magnitude, infinities among them, give NaN wherever they enter.

    The backward pass reads ``x`` and ``codebook`` as they are then: hand it a copy of a codebook that an EMA step rewrites in between
    (``vq_ema_apply`` writes through raw pointers, which autograd's version check does not see)."""
    temperature = float(temperature)
    if not (temperature > 0.0 and math.isfinite(temperature) and 2.0 / temperature <= _F32_MAX):
        raise ValueError(f"temperature must be positive and finite, and 2 / temperature in float32 too, got {temperature}")
    x, cb = _f32_param(x, "x"), _f32_param(codebook, "codebook").contiguous()
    if cb.dim() != 2 or cb.numel() == 0:
        raise ValueError("codebook must be a non-empty [K, D] tensor")
    K, D = cb.shape
    if x.dim() != (3 if channel_major else 2):
        raise ValueError("x must be [B, D, S] with channel_major" if channel_major else "x must be [N, D]")
    if x.shape[1] != D:
        raise ValueError(f"input dim {x.shape[1]} != codebook dim {D}")
    ee = None
    if e_sqnorm is not None:
        ee = _lib.dev_f32(e_sqnorm.detach() if isinstance(e_sqnorm, torch.Tensor) else e_sqnorm)
        if ee.numel() != K:
            raise ValueError(f"e_sqnorm has {ee.numel()} entries, the codebook {K}")
    if channel_major:
        if torch.is_grad_enabled() and (x.requires_grad or cb.requires_grad):
            x = x.permute(0, 2, 1).reshape(-1, D)
        else:
            from .quantizer import _pitched_rows
            x, cb = _pitched_rows(x.detach()), cb.detach()
            B, _, S = x.shape
            out = torch.empty((B * S, K), dtype=torch.float32, device=x.device)
            if out.numel():
                _lib.check(_lib.load().lbm_code_logits_f32(_lib.ptr(x), x.stride(1) if B * D > 1 else S, _lib.VQ_CHANNEL_MAJOR, S,
                                                           _lib.ptr(cb), _lib.ptr(ee), _lib.ptr(out), K, B * S, D, K, temperature,
                                                           _lib.stream_ptr()), "lbm_code_logits_f32")
            return out
    return _CodeLogits.apply(*_rows(x), cb, ee, temperature)


# -------------------------------------------------------------------------------------------------------------- balance
def _score_rows(scores: torch.Tensor, what: str):
    """[..., K] scores as rows the kernels address: (tensor [N, K] with unit stride along K, row stride)."""
    if not isinstance(scores, torch.Tensor):
        raise ValueError(f"{what}: scores must be a tensor")
    if scores.dtype not in _lib.SCORE_TYPES:
        raise ValueError(f"{what}: scores must be float32, float16 or bfloat16, got {scores.dtype}")
    if scores.dim() < 1 or scores.shape[-1] < 1:
        raise ValueError(f"{what}: scores must be [..., K] with K >= 1")
    s = scores if scores.dim() == 2 else scores.reshape(-1, scores.shape[-1])
    N, K = s.shape
    if K > 1 and s.stride(1) != 1:
        s = s.contiguous()
    return s, (s.stride(0) if N > 1 else K)


class _CodeBalance(torch.autograd.Function):
    # Host time counts at training sizes (the kernels take some 60 us): one device check, as few allocations as the lifetimes allow.
    @staticmethod
    def forward(ctx, scores, ld, codes, slots, keep):
        N, K = scores.shape
        dev = scores.device
        lib = _lib.load()
        nbytes = lib.lbm_code_balance_workspace_bytes(N, K)
        if nbytes == 0:
            raise NotImplementedError(f"code_balance_loss supports K <= 8192 (got K={K})")
        sp = _lib.ptr(scores)                        # checks the device; codes and keep were moved to it
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        mean = torch.empty((K,), dtype=torch.float32, device=dev)
        counts = torch.empty((K,), dtype=torch.int64, device=dev)
        saved = torch.empty((2 + N,), dtype=torch.float64, device=dev)      # totals, then (maximum, 1 / sum) of each row
        at = saved.data_ptr()
        _lib.check(lib.lbm_code_balance(sp, _lib.SCORE_TYPES[scores.dtype], ld, None if codes is None else codes.data_ptr(), slots,
                                        None if keep is None else keep.data_ptr(), loss.data_ptr(), counts.data_ptr(), mean.data_ptr(),
                                        at + 16, at, ws.data_ptr(), N, K, _lib.stream_ptr()), "lbm_code_balance")
        ctx.save_for_backward(scores, saved, counts)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts, mean

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, _g_counts, g_mean):
        scores, saved, counts = ctx.saved_tensors
        (N, K), (ld, unit) = scores.shape, scores.stride()
        if K > 1 and unit != 1:              # saved tensors come back in any layout from hooks that offload them
            scores, ld = scores.contiguous(), K
        saved, counts = saved.contiguous(), counts.contiguous()
        ds = torch.empty((N, K), dtype=scores.dtype, device=scores.device)
        if g_mean is not None:
            g_mean = g_mean.contiguous()
        at = saved.data_ptr()
        _lib.check(_lib.load().lbm_code_balance_grad(_lib.ptr(scores), _lib.SCORE_TYPES[scores.dtype], ld, at + 16, counts.data_ptr(), at,
                                                     None if g_loss is None else g_loss.data_ptr(),
                                                     None if g_mean is None else g_mean.data_ptr(), ds.data_ptr(), N, K, _lib.stream_ptr()),
                   "lbm_code_balance_grad")
        return ds, None, None, None, None


@_lib.on_tensor_device
def code_balance_loss(scores: torch.Tensor, codes: torch.Tensor = None, keep: torch.Tensor = None):
    """Usage balance over rows of scores: ``(loss, counts, mean_probs)``.

    With p = softmax(scores) over the last dimension, over the M rows that count: ``mean_probs[k]`` = mean of p[., k] (float32 [K]),
    ``counts[k]`` = how often code k was picked (int64 [K]), ``loss = K * sum_k counts[k] / sum(counts) * mean_probs[k]`` (float32 scalar: 1
    where use is even, up to K where one code takes everything).  Differentiable in ``scores`` through ``loss`` and ``mean_probs`` (an entropy
    of the latter, say); counts are constants.

    ``scores``: [..., K] float32, float16 or bfloat16 (K <= 8192).  ``codes``: integer [...] or [..., slots], the picks of each row (several for
    routers that pick several; negative ones, as ``sample_codes`` answers for empty rows, and ones >= K are not counted); without them the
    best score counts, lowest index first.  ``keep``: bool [...], rows to count (the pipeline's artifact mask, padding); the others' scores are
    not read and their gradient is 0.  A row of nothing but -inf does not count either.  Where no row counts everything is 0.
    Probabilities below the smallest normal float, 2^-126, are 0."""
    s, ld = _score_rows(scores, "code_balance_loss")
    lead = tuple(scores.shape[:-1])
    N = s.shape[0]
    slots = 0
    if codes is not None:
        if codes.is_floating_point() or codes.dtype == torch.bool:
            raise ValueError("code_balance_loss: codes must be integers")
        if tuple(codes.shape) == lead:
            slots = 1
        elif tuple(codes.shape[:-1]) == lead and codes.shape[-1] >= 1:
            slots = int(codes.shape[-1])
        else:
            raise ValueError(f"code_balance_loss: codes {tuple(codes.shape)} do not fit scores {tuple(scores.shape)}")
        codes = codes.to(device=s.device, dtype=torch.int64).contiguous()
    if keep is not None:
        if keep.dtype not in (torch.bool, torch.uint8) or tuple(keep.shape) != lead:
            raise ValueError(f"code_balance_loss: keep must be a bool tensor of shape {lead}")
        keep = keep.to(device=s.device).contiguous().view(torch.uint8)
    return _CodeBalance.apply(s, ld, codes, slots, keep)


# ------------------------------------------------------------------------------------------------------------- sampling
@dataclass
class CodeSampling:
    """Settings of a draw (``sample_codes``), for ``VQVAE.encode(sampling=...)``.  The temperature is that of ``exp(-distance / T)``.
    Each is a number or a tensor with one per code position [B, L//4]; ``allowed``: bool [K] or [B, L//4, K]."""
    temperature: Union[float, torch.Tensor] = 1.0
    top_k: Union[int, torch.Tensor] = 0
    top_p: Union[float, torch.Tensor] = 1.0
    min_p: Union[float, torch.Tensor] = 0.0
    allowed: Optional[torch.Tensor] = None


def _setting(value, name, lead, device, dtype, lo, hi):
    """(per-row tensor or None, value): a number is checked here, a tensor has one entry per row and is read on the device."""
    if isinstance(value, torch.Tensor) and value.dim() > 0:
        if tuple(value.shape) != lead:
            raise ValueError(f"sample_codes: {name} must be a number or a tensor of shape {lead}, got {tuple(value.shape)}")
        if dtype is torch.int32 and (value.is_floating_point() or value.dtype == torch.bool):
            raise ValueError(f"sample_codes: {name} must be integers")
        if dtype is torch.int32 and value.dtype == torch.int64:
            value = value.clamp(-1, 2 ** 31 - 1)
        return value.to(device=device, dtype=dtype).contiguous(), 0
    v = int(value) if dtype is torch.int32 else float(value)
    if dtype is torch.int32 and v != value:
        raise ValueError(f"sample_codes: {name} must be an integer")
    if not (lo <= v <= hi):
        raise ValueError(f"sample_codes: {name} = {value} is outside [{lo}, {hi}]")
    return None, (min(v, 2 ** 31 - 1) if dtype is torch.int32 else v)


@torch.no_grad()
@_lib.on_tensor_device
def sample_codes(scores: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, allowed: torch.Tensor = None,
                 hist: torch.Tensor = None) -> torch.Tensor:
    """One code per row of ``scores`` [..., K], drawn with the uniform numbers ``u`` [...] of [0, 1): int64 [...].

    Weights are exp((s - max s) / ``temperature``) in 64 bits.  ``top_k`` > 0 keeps the k best scores (equal ones: lowest index first);
    ``top_p`` < 1 then keeps, in descending order, every code before which less than that share of the kept weight lies; ``min_p`` then keeps
    codes of at least that share of the best code's weight; the answer is the first index whose running sum exceeds u times the total.
    ``temperature`` 0 answers the best code, lowest index first.  Each setting is a number, or a tensor [...] with one per row (on the
    device, unchecked: temperatures that are not positive mean 0, top_k <= 0 and top_p >= 1 mean all codes).  ``u`` and settings per row
    are taken as float32.

    ``scores``: float32, float16 or bfloat16.  ``allowed``: bool [K] or [..., K], codes that may be drawn.  Scores of +inf share all
    the weight, NaN counts as -inf; a row with nothing to draw from answers -1.  ``hist`` ([K] int64, K <= 32768) is ADDED to when given."""
    s, ld = _score_rows(scores, "sample_codes")
    lead = tuple(scores.shape[:-1])
    N, K = s.shape
    dev = s.device
    if not isinstance(u, torch.Tensor) or not u.is_floating_point() or tuple(u.shape) != lead:
        raise ValueError(f"sample_codes: u must be a floating-point tensor of shape {lead}")
    if u.dtype is torch.float64:
        u = torch.where(u < 1.0, u.clamp(max=1.0 - 2.0 ** -24), u)        # numbers below 1 stay there when they are rounded to fp32
    u = u.to(device=dev, dtype=torch.float32).contiguous()
    t_row, t = _setting(temperature, "temperature", lead, dev, torch.float32, 0.0, math.inf)
    k_row, k = _setting(top_k, "top_k", lead, dev, torch.int32, 0, math.inf)
    p_row, p = _setting(top_p, "top_p", lead, dev, torch.float32, 0.0, 1.0)
    m_row, m = _setting(min_p, "min_p", lead, dev, torch.float32, 0.0, 1.0)
    allowed_ld = 0
    if allowed is not None:
        if allowed.dtype not in (torch.bool, torch.uint8):
            raise ValueError("sample_codes: allowed must be a bool tensor")
        if tuple(allowed.shape) == (K,):
            allowed_ld = 0
        elif tuple(allowed.shape) == tuple(scores.shape):
            allowed_ld = K
        else:
            raise ValueError(f"sample_codes: allowed must be [{K}] or {tuple(scores.shape)}, got {tuple(allowed.shape)}")
        allowed = allowed.to(device=dev).contiguous().view(torch.uint8)
    if hist is not None and (hist.dtype != torch.int64 or hist.numel() != K or not hist.is_contiguous()):
        raise ValueError("hist must be a contiguous int64 tensor of K entries")
    out = torch.empty((N,), dtype=torch.int64, device=dev)
    _lib.check(_lib.load().lbm_code_sample(_lib.ptr(s), _lib.SCORE_TYPES[s.dtype], ld, _lib.ptr(u), _lib.ptr(t_row), t, _lib.ptr(k_row), k,
                                           _lib.ptr(p_row), p, _lib.ptr(m_row), m, _lib.ptr(allowed), allowed_ld, _lib.ptr(out),
                                           _lib.ptr(hist), N, K, _lib.stream_ptr()), "lbm_code_sample")
    return out.reshape(lead)
