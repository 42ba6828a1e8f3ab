"""The operator custom calls in float64: attention and row writes over a paged
key-value cache, the residual norm and token log probabilities, with the
gradients of the last two. Arrays are float64 (or integers) and results are
not rounded, but for the 8-bit rows.

The reference has none of these operators; the definitions are those of
pjrtx_amd/hlo.py's methods of the same names."""
from __future__ import annotations

import numpy as np


def paged_attention(q, k_pages, v_pages, table, lengths, scale=None, window=0):
    """q [B, Hq, D], pages [P, Hkv, S, D], table [B, M], lengths [B]."""
    B, Hq, D = q.shape
    P, Hkv, S, _ = k_pages.shape
    M = table.shape[1]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out = np.zeros((B, Hq, D))
    for b in range(B):
        n = min(max(int(lengths[b]), 0), M * S)
        lo = max(0, n - window) if window else 0
        keys = [j for j in range(lo, n) if 0 <= table[b, j // S] < P]
        if not keys:
            continue
        for h in range(Hq):
            kh = h // (Hq // Hkv)
            k = np.stack([k_pages[table[b, j // S], kh, j % S] for j in keys])
            v = np.stack([v_pages[table[b, j // S], kh, j % S] for j in keys])
            s = scale * (k @ q[b, h])
            e = np.exp(s - s.max())
            out[b, h] = e @ v / e.sum()
    return out


def paged_append(k_pages, v_pages, k_new, v_new, slots):
    k, v = k_pages.copy(), v_pages.copy()
    P, _, S, _ = k.shape
    for n, slot in enumerate(int(x) for x in slots):
        if 0 <= slot < P * S:
            k[slot // S, :, slot % S] = k_new[n]
            v[slot // S, :, slot % S] = v_new[n]
    return k, v


def add_rms_norm(x, residual, gain, eps):
    """(y, t) of rows x [..., D]."""
    t = x if residual is None else x + residual
    return t / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * gain, t


def add_rms_norm_grad(dy, dsum, t, gain, eps):
    r = 1.0 / np.sqrt((t * t).mean(-1, keepdims=True) + eps)
    n, dn = t * r, dy * gain
    dx = r * (dn - n * (dn * n).mean(-1, keepdims=True)) + (0.0 if dsum is None else dsum)
    return dx, (dy * n).reshape(-1, t.shape[-1]).sum(0)


def token_logprobs(logits, tokens, top_k=0):
    m = logits.max(1, keepdims=True)
    e = np.exp(logits - m)
    z = e.sum(1)
    lse = m[:, 0] + np.log(z)
    d = np.where(e > 0, logits - m, 0.0)
    entropy = np.log(z) - (e * d).sum(1) / z
    rows = np.arange(logits.shape[0])
    known = (tokens >= 0) & (tokens < logits.shape[1])
    lp = np.where(known, (logits[rows, np.where(known, tokens, 0)] - m[:, 0]) - np.log(z), 0.0)
    if not top_k:
        return lp, entropy, lse
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
    return lp, entropy, lse, (logits[rows[:, None], ids] - m) - np.log(z)[:, None], ids


def token_logprobs_grad(logits, tokens, lse, entropy, d_lp, d_entropy):
    p = np.exp(logits - lse[:, None])
    logp = np.where(p > 0, logits - lse[:, None], 0.0)
    known = (tokens >= 0) & (tokens < logits.shape[1])
    g = np.where(known, d_lp, 0.0)
    dx = -p * (g[:, None] + d_entropy[:, None] * (logp + entropy[:, None]))
    rows = np.arange(logits.shape[0])[known]
    dx[rows, tokens[known]] += g[known]
    return dx
