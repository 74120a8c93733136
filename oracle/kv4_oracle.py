"""CPU restatement of the 4-bit K/V cache operators (numpy; parity unpinned:
the reference has no counterpart).

Rows are quantised in fp32 exactly as the format says, so codes, lows and steps
can be compared to the bit; values and attention are in 64 bits.
"""
from __future__ import annotations

import numpy as np

GROUP = 32
LIMIT = np.float32(65504.0)


def groups(head_size: int) -> int:
    return -(-head_size // GROUP)


def quantise(rows: np.ndarray):
    """rows [..., d] (any float type) -> code [..., d] uint8, low and step
    [..., groups] float16."""
    x = np.asarray(rows, dtype=np.float32)
    d = x.shape[-1]
    code = np.zeros(x.shape, dtype=np.uint8)
    low = np.zeros((*x.shape[:-1], groups(d)), dtype=np.float16)
    step = np.zeros_like(low)
    with np.errstate(all="ignore"):
        x = np.where(np.isnan(x), x, np.clip(x, -LIMIT, LIMIT)).astype(np.float32)
        for g in range(groups(d)):
            part = x[..., g * GROUP:(g + 1) * GROUP]
            lo, hi = part.min(-1), part.max(-1)  # (numpy's propagate NaN)
            low[..., g] = lo.astype(np.float16)
            step[..., g] = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
            lf, sf = low[..., g].astype(np.float32)[..., None], step[..., g].astype(np.float32)[..., None]
            q = np.rint((part - lf) * (np.float32(1.0) / sf))
            q = np.where(sf > 0, np.clip(q, 0, 15), 0)
            code[..., g * GROUP:(g + 1) * GROUP] = q.astype(np.uint8)
    return code, low, step


def split(code, low, step):
    """(step * code, low) per channel in 64 bits: their sum is the value."""
    d = code.shape[-1]
    st = np.repeat(step.astype(np.float64), GROUP, axis=-1)[..., :d]
    lo = np.repeat(low.astype(np.float64), GROUP, axis=-1)[..., :d]
    return st * code, lo


def stored(rows: np.ndarray) -> np.ndarray:
    """The values that rows are stored as, in 64 bits."""
    a, lo = split(*quantise(rows))
    return a + lo


def attention(q, k_rows, v_rows, scale, num_kv_heads):
    """One sequence: q [H, d], k_rows / v_rows [L, KVH, d] as written ->
    (out [H, d], size [H, d], spread [H]) in 64 bits.  `size` is
    sum_t p_t (step * code + |low|) of V, what rounding a weight is relative
    to; `spread` the largest scale * sum_c |q_c| (step * code + |low|) of a K
    row, what the rounding of a score is relative to."""
    H, d = q.shape
    L = k_rows.shape[0]
    out, size, spread = np.zeros((H, d)), np.zeros((H, d)), np.zeros(H)
    if L == 0:
        return out, size, spread
    G = H // num_kv_heads
    ka, kl = split(*quantise(k_rows))
    va, vl = split(*quantise(v_rows))
    q = q.astype(np.float64)
    for h in range(H):
        kh = h // G
        s = (ka[:, kh] + kl[:, kh]) @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ (va[:, kh] + vl[:, kh])
        size[h] = p @ (va[:, kh] + np.abs(vl[:, kh]))
        spread[h] = abs(scale) * ((ka[:, kh] + np.abs(kl[:, kh])) @ np.abs(q[h])).max()
    return out, size, spread
