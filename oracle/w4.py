"""4-bit weights with group scales in exact arithmetic — test infrastructure (no reference counterpart).

The rules: per row and group s = bf16(absmax / 7), 1 where that is 0; q = clamp(rint(w / s), -7, 7) with the fp32
quotient, ties to even; y = act(sum x q s + bias).
"""
from __future__ import annotations

import numpy as np

from oracle.common import bf16_round


def quantize(w: np.ndarray, group: int) -> tuple[np.ndarray, np.ndarray]:
    """fp32 values of a bf16 matrix `(N, K)` -> integers `(N, K)` and scales `(N, K // group)`, both float64."""
    w = np.asarray(w, np.float32).reshape(len(w), -1, group)
    s = bf16_round(np.abs(w).max(-1) / np.float32(7)).astype(np.float32)
    s = np.where(s == 0, np.float32(1), s)
    q = np.clip(np.rint(w / s[..., None]), -7, 7)
    return q.reshape(len(w), -1).astype(np.float64), s.astype(np.float64)


def pack(q: np.ndarray, s: np.ndarray, group: int) -> tuple[np.ndarray, np.ndarray]:
    """The two arrays of hb_quant_w4's documented layout, word by word: bytes and scale values."""
    n, k = q.shape
    tiles, blocks = -(-n // 16), -(-k // 128)
    words = np.full((tiles, blocks, 256), 0x88888888, np.uint32)
    scales = np.zeros((tiles, blocks, 128 // group, 16))
    for row in range(n):
        for kk in range(0, k, 8):
            word = 0
            for pos, i in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
                word |= (int(q[row, kk + i]) + 8) << (4 * pos)
            r, c = row % 16, kk % 128
            at = 512 * (r // 8) + 64 * (r % 8) + 16 * ((c % 32) // 8) + 4 * (c // 32)
            words[row // 16, kk // 128, at // 4] = word
        for g in range(k // group):
            scales[row // 16, g * group // 128, g % (128 // group), row % 16] = s[row, g]
    return words.view(np.uint8).reshape(tiles, blocks, 1024), scales


def linear(x: np.ndarray, w: np.ndarray, bias, silu: bool, unit: float) -> tuple[np.ndarray, np.ndarray]:
    """`(y, tol)`: y in float64 from the matrix w the weights stand for; tol covers fp32 sums of K products and a
    bias (2^-23 of the absolute sum per addition), SiLU's slope (at most 1.1) and the rounding to 16 bits."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    tol = (x.shape[1] + 1) * 2.0 ** -23 * mag
    if silu:
        with np.errstate(over="ignore"):
            y = y / (1 + np.exp(-y))
        tol = 1.1 * tol + 2.0 ** -20 * np.abs(y)
    return y, tol + unit * (np.abs(y) + tol) + 1e-38
