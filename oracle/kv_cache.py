"""Oracle: the paged key / value cache (rows quantised as they are written, read back) and the attention
over it, in float64.

Test infrastructure only (the tests compare the GPU results against it).
"""
from __future__ import annotations

import numpy as np

TOP = {"bf16": 120, "fp16": 8}     # the exponent at which 256 times the scale exceeds the type's largest value


def grid_e4m3(x):
    """Rounded to the e4m3 grid (1.xxx * 2^e, e >= -6; steps of 2^-9 below), ties to even; no range limit."""
    x = np.asarray(x, np.float64)
    e = np.frexp(x)[1]
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    with np.errstate(invalid="ignore"):
        return np.where(np.isfinite(x), np.rint(x / step) * step, x)


def quantise(rows, dtype):
    """rows [..., D] -> (e4m3 values, exponents E): the least E >= -126 with amax <= 448 * 2^E over the finite
    elements; NaN and infinities become NaN."""
    x = np.asarray(rows, np.float64)
    fin = np.isfinite(x)
    amax = np.abs(np.where(fin, x, 0.0)).max(-1)
    E = np.full(amax.shape, -126)
    for idx in np.ndindex(amax.shape):
        while amax[idx] > 448.0 * 2.0 ** E[idx]:
            E[idx] += 1
    q = grid_e4m3(np.where(fin, x, 0.0) * np.ldexp(1.0, -E)[..., None])
    most = np.where(E == TOP[dtype], 240.0, 448.0)[..., None]
    return np.where(fin, np.clip(q, -most, most), np.nan), E


def attention(q, k, v, lens, cu, scale, causal=True):
    """q [T, H, D]; k, v: per sequence [len, Hkv, D] -> (out [T, H, D], lse [H, T], weight [T, H, D], reach [H, T]):
    weight = sum_j p_j |v_j| and reach = the largest |scale| sum |q| |k| of a visible token, for error bounds.
    Rows of no sequence: NaN."""
    T, H, D = q.shape
    out, weight = np.full((T, H, D), np.nan), np.zeros((T, H, D))
    lse, reach = np.full((H, T), np.nan), np.zeros((H, T))
    for s, L in enumerate(lens):
        n = cu[s + 1] - cu[s]
        for i in range(n):
            t = cu[s] + i
            vis = max(0, min(L, L - n + i + 1)) if causal else L
            for h in range(H):
                hk = h * k[s].shape[1] // H
                if vis == 0:
                    out[t, h], lse[h, t] = 0.0, -np.inf
                    continue
                x = scale * (k[s][:vis, hk] @ q[t, h])
                m = x.max()
                p = np.exp(x - m)
                out[t, h] = p @ v[s][:vis, hk] / p.sum()
                weight[t, h] = p @ np.abs(v[s][:vis, hk]) / p.sum()
                lse[h, t] = m + np.log(p.sum())
                reach[h, t] = abs(scale) * (np.abs(k[s][:vis, hk]) @ np.abs(q[t, h])).max()
    return out, lse, weight, reach
