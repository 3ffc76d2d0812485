"""What the code-score operators are measured on: cases, inputs, the plain forms and the 64-bit definitions.

Operators (rows = code positions of encoded epochs, K = codes of the VQ-VAE's codebook):

  logits   code_logits        scores[n, k] = (2 x_n.e_k - |e_k|^2) / T, and the gradients of x and of the codebook
  balance  code_balance_loss  usage-balance loss, codes per row counted, mean probabilities; and the gradient of the scores
  sample   sample_codes       one code per row from given uniform numbers: temperature, top-k, top-p, min-p

Sizes: 375 rows are one 30-channel 3 s epoch at 500 Hz (1500 samples, four samples per code), 64 epochs are the training batch,
512 codes of 256 values the shipped codebook; 2500 rows are one 10 s epoch at 1 kHz, searched against 8192 codes.
"""
import math

import torch

own = False      # False: plain torch forms; True: this package's operators

S_EPOCH = 375        # codes of one 1500-sample epoch
S_LONG = 2500        # codes of one 10 000-sample epoch
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one epoch scored as it arrives: latency
        {"name": "logits_one_epoch", "op": "logits", "N": S_EPOCH, "D": 256, "K": 512, "train": False, "T": 0.1},
        # the quantizer's training step on the reference's batch of 64 epochs
        {"name": "logits_batch_train", "op": "logits", "N": 64 * S_EPOCH, "D": 256, "K": 512, "train": True, "T": 0.1},
        # odd sizes: the shipped codebook without its repeated rows, a narrow latent, a ragged batch
        {"name": "logits_odd_train", "op": "logits", "N": 5003, "D": 100, "K": 413, "train": True, "T": 0.25},
        # 16 long epochs against the large codebook
        {"name": "logits_large_codebook", "op": "logits", "N": 16 * S_LONG, "D": 256, "K": 8192, "train": False, "T": 0.1},
        # the training batch: loss, counts, mean probabilities and the scores' gradient
        {"name": "balance_batch_train", "op": "balance", "N": 64 * S_EPOCH, "K": 512, "type": "f32", "slots": 1, "keep": 1.0,
         "train": True},
        # a small head under autocast, no codes given (the best score counts), a tenth of the rows rejected
        {"name": "balance_small_bf16", "op": "balance", "N": 4 * S_EPOCH + 1, "K": 61, "type": "bf16", "slots": 0, "keep": 0.9,
         "train": True},
        # usage of a whole chunk of 4096 epochs, no gradient
        {"name": "balance_chunk", "op": "balance", "N": 4096 * S_EPOCH, "K": 512, "type": "f32", "slots": 1, "keep": 0.95,
         "train": False},
        # the large codebook, two codes per row, padded rows
        {"name": "balance_large_codebook_bf16", "op": "balance", "N": 16 * S_LONG, "K": 8192, "type": "bf16", "slots": 2,
         "keep": 0.8, "train": True},
        # one epoch, every filter on: latency
        {"name": "sample_one_epoch", "op": "sample", "N": S_EPOCH, "K": 512, "type": "f32", "per_row": False, "T": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.02},
        # 24 generated sequences at one position, each with its own settings, large vocabulary of codes
        {"name": "sample_step_bf16", "op": "sample", "N": 24, "K": 8192, "type": "bf16", "per_row": True, "T": 1.0,
         "top_k": 200, "top_p": 0.9, "min_p": 0.01},
        # a chunk of 1024 epochs tokenized by sampling, temperature and nucleus
        {"name": "sample_chunk", "op": "sample", "N": 1024 * S_EPOCH, "K": 512, "type": "f32", "per_row": False, "T": 1.0,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # long epochs, large codebook, top-k before the nucleus
        {"name": "sample_large_codebook_f16", "op": "sample", "N": 16 * S_LONG, "K": 8192, "type": "f16", "per_row": False,
         "T": 1.3, "top_k": 100, "top_p": 0.95, "min_p": 0.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logits", "balance", "sample"])
    if op == "logits":
        train = rng.random() < 0.5
        K, D = _log_int(rng, 16, 8192), rng.choice([8, 32, 64, 100, 128, 200, 255, 256])
        N = _log_int(rng, 1, max(1, min(1_500_000, 320_000_000 // K, 160_000_000_000 // ((6 if train else 2) * K * D))))
        return {"op": op, "N": N, "D": D, "K": K, "train": train, "T": rng.choice([0.05, 0.1, 0.3, 1.0])}
    K = _log_int(rng, 2, 8192)
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "balance":
        N = _log_int(rng, 1, max(1, min(1_500_000, 320_000_000 // K)))
        return {"op": op, "N": N, "K": K, "type": kind, "slots": rng.choice([0, 1, 1, 2, 4]),
                "keep": rng.choice([1.0, 0.95, 0.5]), "train": rng.random() < 0.6}
    N = _log_int(rng, 1, max(1, min(384_000, 190_000_000 // K)))
    return {"op": op, "N": N, "K": K, "type": kind, "per_row": rng.random() < 0.3, "T": rng.choice([0.3, 0.7, 1.0, 1.5]),
            "top_k": rng.choice([0, 1, 20, 100, 1000]), "top_p": rng.choice([1.0, 0.5, 0.9, 0.99]),
            "min_p": rng.choice([0.0, 0.0, 0.01, 0.1])}


# ----------------------------------------------------------------------------------------------------------------- inputs
def _latents(g, N, D, K):
    """Encoder outputs round codes that are used unevenly, as a trained codebook's are: norms near one, noise of a few tenths."""
    e = torch.randn((K, D), generator=g, device="cuda") / math.sqrt(D)
    used = (torch.rand((N,), generator=g, device="cuda") ** 3 * K).long().clamp_(max=K - 1)
    x = e[used] + torch.randn((N, D), generator=g, device="cuda") * (0.5 / math.sqrt(D))
    return x, e


def _scores(g, N, K, dtype):
    """Scores as code_logits makes them from such latents (64 values wide: only the scores matter here), in the given type."""
    x, e = _latents(g, N, 64, K)
    s = (2.0 * (x @ e.t()) - (e * e).sum(1)) / 0.1
    return s.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    N, K = case["N"], case["K"]
    st = {"case": case}
    if case["op"] == "logits":
        st["x"], st["e"] = _latents(g, N, case["D"], K)
        if case["train"]:
            st["g"] = torch.randn((N, K), generator=g, device="cuda") / N
        return st
    st["s"] = _scores(g, N, K, TYPES[case["type"]])
    if case["op"] == "balance":
        slots = case["slots"]
        st["codes"] = None
        if slots:      # the codes that the router picked: the best scores, as indices
            st["codes"] = st["s"].argmax(1) if slots == 1 else st["s"].topk(min(slots, K), dim=1).indices.contiguous()
        st["keep"] = None if case["keep"] >= 1.0 else torch.rand((N,), generator=g, device="cuda") < case["keep"]
        if st["keep"] is not None:      # rows of rejected epochs hold whatever the padding left there
            st["s"][~st["keep"]] = float("nan")
        st["g_loss"] = torch.tensor(0.01, device="cuda")
        st["g_mean"] = torch.randn((K,), generator=g, device="cuda") * 0.01
        return st
    st["u"] = torch.rand((N,), generator=g, device="cuda")
    names = ("T", "top_k", "top_p", "min_p")
    if case["per_row"]:     # each row its own request: settings spread round the case's
        r = torch.rand((4, N), generator=g, device="cuda")
        st["T"] = torch.where(r[0] < 0.1, torch.zeros_like(r[0]), case["T"] * (0.5 + r[0]))      # a tenth of them greedy
        st["top_k"] = (case["top_k"] * 2 * r[1]).to(torch.int32)
        st["top_p"] = (case["top_p"] + (1 - case["top_p"]) * (2 * r[2] - 1)).clamp(max=1.0)
        st["min_p"] = case["min_p"] * 2 * r[3]
    else:
        for n in names:
            st[n] = case[n]
    return st


# ------------------------------------------------------------------------------------------------------------------- runs
def run(state):
    case = state["case"]
    return {"logits": _run_logits, "balance": _run_balance, "sample": _run_sample}[case["op"]](state, case)


def _run_logits(st, case):
    x, e, T = st["x"], st["e"], case["T"]
    if own:
        import lbm_amd
        if not case["train"]:
            return lbm_amd.code_logits(x, e, temperature=T)
        xg, eg = x.detach().requires_grad_(), e.detach().requires_grad_()
        s = lbm_amd.code_logits(xg, eg, temperature=T)
        dx, de = torch.autograd.grad(s, (xg, eg), st["g"])
        return {"logits": s.detach(), "dx": dx, "de": de}
    s = ((x @ e.t()) * 2.0 - (e * e).sum(1)) / T
    if not case["train"]:
        return s
    g = st["g"]
    dx = (g @ e) * (2.0 / T)
    de = (g.t() @ x - g.sum(0)[:, None] * e) * (2.0 / T)
    return {"logits": s, "dx": dx, "de": de}


def _run_balance(st, case):
    s, codes, keep = st["s"], st["codes"], st["keep"]
    if own:
        import lbm_amd
        if not case["train"]:
            loss, counts, mean = lbm_amd.code_balance_loss(s, codes, keep=keep)
            return {"loss": loss, "counts": counts, "mean": mean}
        sg = s.detach().requires_grad_()
        loss, counts, mean = lbm_amd.code_balance_loss(sg, codes, keep=keep)
        (ds,) = torch.autograd.grad((loss, mean), (sg,), (st["g_loss"], st["g_mean"]))
        return {"loss": loss.detach(), "counts": counts, "mean": mean.detach(), "ds": ds}
    N, K = s.shape
    v = s.float()
    if keep is not None:
        v = torch.where(keep[:, None], v, torch.zeros((), device=v.device))
    p = torch.exp(v - v.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    kept = torch.ones((N,), device=s.device) if keep is None else keep.float()
    rows = kept.sum().clamp(min=1.0)
    mean = (p.double() * kept[:, None]).sum(0).div(rows).float() if N > 65536 else (p * kept[:, None]).sum(0) / rows
    if codes is None:
        top = torch.where(v == v.amax(1, keepdim=True), torch.arange(K, device=s.device), K).amin(1)      # lowest index of the best
        codes = top
    picked = codes.reshape(N, -1)
    counts = torch.zeros((K,), dtype=torch.int64, device=s.device)
    counts.index_add_(0, picked.reshape(-1), kept.long()[:, None].expand_as(picked).reshape(-1))
    f = counts.float() / counts.sum().clamp(min=1)
    loss = K * (f * mean).sum()
    if not case["train"]:
        return {"loss": loss, "counts": counts, "mean": mean}
    # p (a - sum p a) with a taken relative to its value at the row's best score: where one p is near one, the plain difference cancels
    a = (st["g_loss"].double() * K * (counts.double() / counts.sum().clamp(min=1)) + st["g_mean"].double()).float()
    a = a - a[v.argmax(1)][:, None]
    ds = p * (a - (p * a).sum(1, keepdim=True)) * (kept / rows)[:, None]
    return {"loss": loss, "counts": counts, "mean": mean, "ds": ds.to(s.dtype)}


def _run_sample(st, case):
    s, u = st["s"], st["u"]
    if own:
        import lbm_amd
        return lbm_amd.sample_codes(s, u, temperature=st["T"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
    # 64 bits: a number next to a border has to fall on the right side of it
    N, K = s.shape
    col = (lambda t: t.double()[:, None]) if case["per_row"] else (lambda t: t)
    T, top_k, top_p, min_p = col(st["T"]), col(st["top_k"]), col(st["top_p"]), col(st["min_p"])
    v = s.double()
    d = v - v.amax(1, keepdim=True)
    if case["per_row"]:
        greedy = T == 0
        w = torch.where(d == 0, 1.0, torch.exp(d / torch.where(greedy, torch.ones_like(T), T)))
    else:
        w = torch.exp(d / T)
    del d
    on = (lambda t, lim: True) if case["per_row"] else (lambda t, lim: 0 < t < lim)
    if on(top_k, K) or on(top_p, 1.0):
        order = torch.sort(v, dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        if case["per_row"]:
            rank = torch.arange(K, device=s.device)
            ws = torch.where((top_k > 0) & (rank >= top_k), 0.0, ws)
        elif 0 < top_k < K:
            ws[:, top_k:] = 0.0
        cum = ws.cumsum(1)
        before = cum - ws
        # a candidate stays while what stands before it is below the share asked for
        stays = (before < top_p * cum[:, -1:]) & (ws > 0)
        if case["per_row"]:
            stays = torch.where(top_p < 1.0, stays, ws > 0)
        elif not top_p < 1.0:
            stays = ws > 0
        stays[:, 0] = True
        w = torch.where(torch.zeros_like(stays).scatter_(1, order, stays), w, 0.0)
        del order, ws, cum, before, stays
    w = torch.where(w >= min_p, w, 0.0)
    cum = w.cumsum(1)
    hit = cum > u.double()[:, None] * cum[:, -1:]
    code = torch.where(hit, torch.arange(K, device=s.device), K).amin(1)
    last = torch.where(w > 0, torch.arange(K, device=s.device), -1).amax(1)
    code = torch.minimum(code, last)
    if case["per_row"]:
        best = torch.where(v == v.amax(1, keepdim=True), torch.arange(K, device=s.device), K).amin(1)
        code = torch.where(greedy[:, 0], best, code)
    return code


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    N, K = case["N"], case["K"]
    if case["op"] == "logits":
        D = case["D"]
        if not case["train"]:
            return {"bytes": 4 * (N * D + K * D + N * K), "flops": 2 * N * K * D}
        return {"bytes": 4 * (2 * N * D + 2 * K * D + 2 * N * K), "flops": 6 * N * K * D}
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "balance":
        rest = N * (8 * case["slots"] + (case["keep"] < 1.0)) + 12 * K
        return {"bytes": N * K * size * (2 if case["train"] else 1) + rest, "flops": N * K * (9 if case["train"] else 4)}
    return {"bytes": N * K * size + N * (12 + (16 if case["per_row"] else 0)), "flops": 8 * N * K}


# ------------------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    st = prepare(case, seed)
    N, K = case["N"], case["K"]
    if case["op"] == "logits":
        x, e, T = st["x"].double(), st["e"].double(), case["T"]
        s = torch.empty((N, K), dtype=torch.float64, device="cuda")
        norm = e.pow(2).sum(1)
        for a in range(0, N, 65536):
            torch.sub(2 * (x[a:a + 65536] @ e.t().contiguous()), norm, out=s[a:a + 65536])
        s /= T
        if not case["train"]:
            return s
        g = st["g"].double()
        # d s[n,k] / d x_n = 2 e_k / T;  d s[n,k] / d e_k = 2 (x_n - e_k) / T
        return {"logits": s, "dx": 2 / T * torch.mm(g, e), "de": 2 / T * (torch.mm(g.t().contiguous(), x) - e * g.sum(0).unsqueeze(1))}
    if case["op"] == "balance":
        rows = torch.arange(N, device="cuda") if st["keep"] is None else st["keep"].nonzero()[:, 0]
        M = max(1, rows.numel())
        step = max(1, 100_000_000 // K)
        mean = torch.zeros((K,), dtype=torch.float64, device="cuda")
        counts = torch.zeros((K,), dtype=torch.int64, device="cuda")
        for a in range(0, rows.numel(), step):
            r = rows[a:a + step]
            v = st["s"][r].double()
            mean += torch.softmax(v, 1).sum(0)
            c = v.max(1, keepdim=True).values.eq(v).int().argmax(1) if st["codes"] is None else st["codes"][r].reshape(-1)
            counts += torch.bincount(c, minlength=K)
        mean /= M
        f = counts.double() / max(1, int(counts.sum()))
        out = {"loss": K * torch.dot(f, mean), "counts": counts, "mean": mean}
        if case["train"]:
            a_k = st["g_loss"].double() * K * f + st["g_mean"].double()
            ds = torch.zeros((N, K), dtype=torch.float64, device="cuda")
            for a in range(0, rows.numel(), step):
                r = rows[a:a + step]
                p = torch.softmax(st["s"][r].double(), 1)
                ds[r] = p * (a_k - p @ a_k[:, None]) / M
            out["ds"] = ds
        return out
    if N * K > 4_000_000:
        return None
    import numpy as np
    s, u = st["s"].double().cpu().numpy(), st["u"].double().cpu().numpy()
    par = {}
    for n in ("T", "top_k", "top_p", "min_p"):
        par[n] = st[n].double().cpu().numpy() if case["per_row"] else np.full((N,), float(st[n]))
    out = np.empty((N,), np.int64)
    for i in range(N):
        if par["T"][i] == 0:
            out[i] = int(np.argmax(s[i]))
            continue
        w = np.exp((s[i] - s[i].max()) / par["T"][i])
        order = np.lexsort((np.arange(K), -s[i]))
        if par["top_k"][i] > 0:
            order = order[:int(par["top_k"][i])]
        if par["top_p"][i] < 1:
            total = math.fsum(w[order])
            before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
            order = order[(before < par["top_p"][i] * total) | (np.arange(order.size) == 0)]
        left = np.sort(order[w[order] >= par["min_p"][i]])
        cum = np.cumsum(w[left])
        out[i] = left[min(int(np.searchsorted(cum, u[i] * cum[-1], side="right")), left.size - 1)]
    return torch.from_numpy(out)
