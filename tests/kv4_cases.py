"""Inputs and tolerances of the 4-bit cache tests."""
from __future__ import annotations

import math

import numpy as np
import torch

from oracle import kv4_oracle as K4

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF_STEP = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}


def rows(n, kvh, d, dtype, seed):
    """CPU rows [n, kvh, d] whose channels differ in size and offset."""
    g = torch.Generator().manual_seed(seed)
    gain = torch.exp(0.5 * torch.randn((kvh, d), generator=g))
    off = 0.5 * torch.randn((kvh, d), generator=g)
    return (torch.randn((n, kvh, d), generator=g) * gain + off).to(DTYPES[dtype])


def np64(t):
    return t.detach().cpu().double().numpy()


def np32(t):
    return t.detach().cpu().float().numpy()


def tables_for(lens, bs, seed, width=0):
    """Block tables of a shuffled pool (-1 past each sequence) and its size."""
    rng = np.random.default_rng(seed)
    need = [-(-n // bs) for n in lens]
    pool = sum(need) + 3
    perm = rng.permutation(pool)
    bt = np.full((len(lens), max([width, 1] + need)), -1, dtype=np.int32)
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        at += n
    return bt, pool


def slots_for(bt, lens, bs):
    """Flat slot of every token, sequence after sequence."""
    out = [bt[s, np.arange(n) // bs].astype(np.int64) * bs + np.arange(n) % bs
           for s, n in enumerate(lens)]
    return np.concatenate(out).astype(np.int32) if out else np.zeros(0, np.int32)


def attention_bound(dtype, out, size, spread):
    """Largest error of an output against 64 bits.

    A score: 32 products per group in fp32, each group's sum scaled and added
    (at most 12 more roundings): under 48 * 2^-24 of the sum of magnitudes; an
    fp32 query in two fp16 parts drops 2^-22 of its largest element, at most
    32 elements of a group at once, under 2^-17 of spread between them in all;
    and the rounded score itself and the exponential, 2^-22 of the spread and
    2^-22.  An error e of the scores moves an output by at most 2e * size.
    A weight p is rounded to fp16 (bf16 output: by 2^-11 of it) or to two fp16
    parts (2^-22), and these weights are the ones that are summed to divide by:
    with p' = p (1 + e), |e| <= u, the quotient sum p' v / sum p' moves by
    sum p e (v - out) / sum p' <= u (size + |out|) <= 2 u size.  Times its step
    it is rounded once more, by the same u of step * code: 3 u size in all.
    And the sum over the tokens adds 2^-20 at most (64 roundings of partial
    sums, several chains).  Then the output's own rounding: half a step of its
    value, and for fp16 at least half of the subnormal unit 2^-24 (an output of
    3e-5 is 2^-15.02 and is held as a multiple of 2^-24, so it is off by up to
    2^-25 whatever computed it)."""
    weight = 3 * (2.0 ** -11 if dtype == "bf16" else 2.0 ** -22)
    e = (2.0 ** -17) * spread[..., None] + 2.0 ** -21
    rounding = np.maximum(HALF_STEP[dtype] * np.abs(out), 2.0 ** -25 if dtype == "fp16" else 0.0)
    return rounding + (weight + 2.0 ** -20 + 2 * e) * size + 1e-30


def reference(q, key, value, lens, scale, kvh, starts=None):
    """Stacked oracle results of a batch: key / value CPU rows of every token,
    sequence after sequence (starts: first row of each)."""
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]]) if starts is None else starts
    r = [K4.attention(np64(q[s]), np32(key[a:a + n]), np32(value[a:a + n]), scale, kvh)
         for s, (a, n) in enumerate(zip(starts, lens))]
    return tuple(np.stack([x[i] for x in r]) for i in range(3))


def scale_of(d):
    return 1.0 / math.sqrt(d)
