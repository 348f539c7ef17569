"""CPU oracle (64 bits) of the serving operators that have no reference counterpart -- test
infrastructure only: adapters of many requests, verification of drafted tokens, and WKV-7 over
drafted tokens.  Each also returns what its tests bound rounding errors with."""
import math

import numpy as np
import torch

FLT_MAX = float(np.finfo(np.float32).max)
U32 = 2.0 ** -24  # half a step of fp32, relative


# ---------------------------------------------------------------- adapters

def lora(x, a, b, base, adapters, scale=None, relu2=False):
    """y [m, n] float64 and a bound of the error of the fp32 computation before the rounding to
    fp16.  The sum over k: every addition rounds its partial sum, whose size is about
    s = sqrt(sum (x a)^2) for terms of random sign, so the errors walk to u s sqrt(k) at most in
    the rms; 8 of those are allowed.  h enters the second product as two fp16 halves of a value
    whose row's largest is at least 2^14: within 2^-22 of itself, and where the second half is a
    denormal, half of 2^-24, which is 2^-39 of that largest; that product's r + 2 roundings count
    u each."""
    x, a, b, y = x.double(), a.double(), b.double(), base.double().clone()
    G, R, K = a.shape
    err = torch.zeros_like(y)
    for i, g in enumerate(adapters.tolist()):
        if g < 0:
            continue
        if g >= G:
            y[i] = math.nan
            continue
        s = 1.0 if scale is None else float(scale[g])
        h = s * (a[g] @ x[i])
        eh = 8 * U32 * math.sqrt(K) * abs(s) * torch.sqrt((a[g] ** 2) @ (x[i] ** 2)) + 2.0 ** -22 * h.abs()
        eh = eh + 2.0 ** -39 * (h.abs().max() if R else 0.0) + 2 * U32 * h.abs()
        y[i] += b[g] @ h
        err[i] = b[g].abs() @ eh + (R + 2) * U32 * (b[g].abs() @ h.abs())
    err = err + U32 * y.abs()
    if relu2:
        pos = torch.where(torch.isnan(y), y, y.clamp(min=0.0))
        err = 2 * pos * err + err * err + U32 * pos * pos
        y = pos * pos
    return y, err


# ---------------------------------------------------------------- verification

def probabilities(logits, temperature=1.0, top_k=-1, top_p=1.0):
    """p (float64) of one row of logits, by distinct logit values."""
    l = np.asarray(logits, dtype=np.float64)
    l = np.clip(np.where(np.isnan(l), 0.0, l), -FLT_MAX, FLT_MAX)
    V = l.size
    if not 0 < top_k <= V:
        top_k = V
    if not 0 <= top_p <= 1:
        top_p = 1.0
    if top_p == 0:
        top_k, top_p = 1, 1.0
    x = np.exp((l - l.max()) / temperature)
    if top_k == V and top_p >= 1.0:
        return x / x.sum()
    vals, inv, cnt = np.unique(-l, return_inverse=True, return_counts=True)  # descending logits
    mass = np.exp((-vals + vals[0]) / temperature) * cnt
    n, m = np.cumsum(cnt), np.cumsum(mass)
    goal = top_p * x.sum()
    big = (n >= top_k) | ((m >= goal) if top_p < 1.0 else np.zeros(n.size, bool))
    i = int(np.argmax(big)) if big.any() else n.size - 1
    share = (top_k - (n[i] - cnt[i])) / cnt[i]
    if top_p < 1.0 and mass[i] > 0:
        share = min(share, (goal - (m[i] - mass[i])) / mass[i])
    part = np.zeros(vals.size)
    part[:i] = 1.0
    part[i] = 1.0 if i == 0 else min(max(share, 0.0), 1.0)
    kept = x * part[inv]
    return kept / kept.sum()


def verify(logits, drafts, uniforms, n_draft=None, draft_probs=None, **filt):
    """tokens [B, K+1], accepted [B] (numpy int32)."""
    B, T, V = logits.shape
    K = T - 1
    tokens, accepted = np.full((B, T), -1, np.int32), np.full(B, -1, np.int32)
    for b in range(B):
        n = K if n_draft is None else int(n_draft[b])
        if not 0 <= n <= K:
            continue
        i = 0
        while True:
            w = probabilities(logits[b, i], **filt)
            if i == n:
                break
            d = int(drafts[b, i])
            known = 0 <= d < V
            pd = w[d] if known else 0.0
            qd = 1.0 if draft_probs is None else (float(draft_probs[b, i, d]) if known else 0.0)
            if not float(uniforms[b, i]) * qd < pd:
                rest = w.copy()
                if draft_probs is not None:
                    rest = np.maximum(rest - draft_probs[b, i].astype(np.float64), 0.0)
                elif known:
                    rest[d] = 0.0
                w = rest if rest.sum() > 0 else w
                break
            tokens[b, i] = d
            i += 1
        c = np.cumsum(w)
        over = c > float(uniforms[b, K]) * c[-1]
        tokens[b, i] = int(np.argmax(over)) if over.any() else int(np.nonzero(w > 0)[0][-1])
        accepted[b] = i
    return tokens, accepted


# ---------------------------------------------------------------- the recurrence over drafts

def wkv_drafts(pool, slots, kept, pending, pending_rows, new, H):
    """(y, y_err, pool, pool_err) in float64: the recurrence, and a running bound of the fp32
    evaluation's error.  Per token, with u = 2^-24: the decay is within 8u of itself (one division
    and two exponentials, whose argument is below 1.3 and so carries 4u into them); a 64-term dot
    product in chains of 8 and three joins rounds each term at most 11 times; the update rounds
    three times, at most the sum of its terms' sizes each."""
    pool = pool.double().clone()
    perr = torch.zeros_like(pool)
    B, T = new["r"].shape[:2]
    y = torch.zeros(B, T, H * 64, dtype=torch.float64)
    yerr = torch.zeros_like(y)

    def vec(src, n, row, t):
        return src[n][row, t].double().view(H, 64)

    def token(S, E, src, row, t):
        w, k, v, a, b = (vec(src, n, row, t) for n in "wkvab")
        d = torch.exp(-math.exp(-0.5) * torch.sigmoid(w))[:, None, :]
        ab, bb, vk = a.abs()[:, None, :], b.abs()[:, None, :], (v.abs()[:, :, None] * k.abs()[:, None, :])
        sa = (S * a[:, None, :]).sum(-1, keepdim=True)
        mag = (S.abs() * ab).sum(-1, keepdim=True)
        ea = (E * ab).sum(-1, keepdim=True) + 11 * U32 * mag
        E2 = E * d + 8 * U32 * S.abs() * d + ea * bb + 3 * U32 * (S.abs() * d + mag * bb + vk)
        return S * d + sa * b[:, None, :] + v[:, :, None] * k[:, None, :], 1.01 * E2

    for i in range(B):
        S, E = pool[slots[i]].clone(), torch.zeros(H, 64, 64, dtype=torch.float64)
        nk = 0 if kept is None else int(kept[i])
        for t in range(nk):
            S, E = token(S, E, pending, int(pending_rows[i]) if pending_rows is not None else i, t)
        if nk:
            pool[slots[i]], perr[slots[i]] = S, E
        for t in range(T):
            S, E = token(S, E, new, i, t)
            r = vec(new, "r", i, t)
            y[i, t] = (S * r[:, None, :]).sum(-1).reshape(-1)
            yerr[i, t] = (E * r.abs()[:, None, :]).sum(-1).reshape(-1) + 11 * U32 * (
                S.abs() * r.abs()[:, None, :]).sum(-1).reshape(-1)
    return y, yerr, pool, perr
