"""Plain context attention in float64 — test infrastructure.

The non-differential `SDPA(q, k, v)` of the reference's cross-attention (dit.py:131-147, 203-215), one query head at
a time over the states that are valid, with shared states in front of a batch element's own, and the bound within
which 16-bit kernels have to stay.
"""
from __future__ import annotations

import numpy as np

EXP2_ERROR = 8e-5  # of the polynomial that takes a share of the exponentials (its fit: 7.5e-5)


def context_attention(q, kv, heads, head_dim, *, kv_heads=None, lens=None, mask=None, shared_kv=None,
                      shared_mask=None, q_weight=None, eps=1e-6, scale=None, unit=2.0 ** -8, floor=0.0):
    """`(out, tol)`, both `(B, Lq, H * D)` float64. `unit` is the 16-bit type's largest relative rounding error, `floor`
    what a weight below the type's normal range may be off by, in units of the row's largest weight.

    tol, element by element, with A = sum_j p_j |v_j|: the output's own rounding (unit |o|), the weights' rounding
    (unit A), scores off by delta (fp32 sums of D products, the normed query's rounding where there is a norm, the
    relative error of the exponentials' polynomial), which moves every weight by at most e^delta above and below
    (e^(2 delta) - 1 times A), and fp32 sums over n keys."""
    kv_heads = kv_heads or heads
    scale = head_dim ** -0.5 if scale is None else scale
    q, kv = np.asarray(q, np.float64), np.asarray(kv, np.float64)
    bsz, lq, _ = q.shape
    lkv = kv.shape[1]
    out, tol = np.zeros_like(q), np.zeros_like(q)
    for b in range(bsz):
        valid = np.ones(lkv, bool)
        if lens is not None:
            valid &= np.arange(lkv) < int(lens[b])
        if mask is not None:
            valid &= np.asarray(mask[b], bool)
        states = kv[b][valid]
        if shared_kv is not None:
            sh = np.asarray(shared_kv, np.float64)
            states = np.concatenate([sh if shared_mask is None else sh[np.asarray(shared_mask, bool)], states])
        n = len(states)
        if n == 0:
            continue
        states = states.reshape(n, 2, kv_heads, head_dim)
        for h in range(heads):
            g = h // (heads // kv_heads)
            k, v = states[:, 0, g], states[:, 1, g]
            cols = slice(h * head_dim, (h + 1) * head_dim)
            x = q[b, :, cols]
            delta = head_dim * 2.0 ** -23
            if q_weight is not None:
                x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(q_weight, np.float64)
                delta += unit + 2.0 ** -20
            s = scale * (x @ k.T)
            delta = delta * scale * (np.abs(x) @ np.abs(k).T).max(-1, keepdims=True) + EXP2_ERROR
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o, a = p @ v, p @ np.abs(v)
            out[b, :, cols] = o
            tol[b, :, cols] = unit * (a + np.abs(o)) * (1 + unit) + np.expm1(2 * delta) * a + n * 2.0 ** -23 * a
            tol[b, :, cols] += floor * p.max(-1, keepdims=True) * np.abs(v).sum(0)
    return out, tol
