"""The 4-bit cache without a GPU: the format's properties on the oracle, and
every refusal of the C entry points and of the Python ones."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as K4
from xllms_amd import _lib
from xllms_amd import kv4_cache as KV4
from xllms_amd.paged_attention import (NXT_ATTN_E_INVALID, NXT_ATTN_E_UNSUPPORTED, NXT_ATTN_OK,
                                       NXT_KV_BF16, NXT_KV_FP16, NXT_KV_FP32)

HEAD_SIZES = (32, 64, 80, 96, 112, 128, 192, 256)


@pytest.mark.parametrize("d", HEAD_SIZES)
@pytest.mark.parametrize("scale", [1e-3, 1.0, 300.0])
def test_values_are_within_half_a_step(d, scale):
    x = (np.random.default_rng(d).standard_normal((50, 3, d)) * scale).astype(np.float32)
    code, low, step = K4.quantise(x)
    err = np.abs(K4.stored(x) - x)
    st = np.repeat(step.astype(np.float64), 32, axis=-1)[..., :d]
    lo = np.repeat(np.abs(low.astype(np.float64)), 32, axis=-1)[..., :d]
    # half a step; the top of the range by the step's rounding (15 codes of
    # 2^-11 of it, or of half a subnormal unit) and the bottom by the low's
    slack = 15 * np.maximum(st * 2.0 ** -11, 2.0 ** -25) + np.maximum(lo * 2.0 ** -11, 2.0 ** -25)
    assert (err <= st * (0.5 + 2.0 ** -18) + slack).all()
    assert code.max() == 15 and code.min() == 0


def test_constant_nan_and_infinite_groups():
    x = np.zeros((5, 1, 64), dtype=np.float32)
    x[0] = 1.5                      # constant: step 0
    x[1, 0, 3] = np.nan             # one NaN: its group only
    x[2, 0, :] = 1.0
    x[2, 0, 40] = np.inf
    x[3, 0, 7] = -np.inf
    x[4] = 1e30
    v = K4.stored(x)
    assert (v[0] == 1.5).all()
    assert np.isnan(v[1, 0, :32]).all() and (v[1, 0, 32:] == 0).all()
    assert abs(v[2, 0, 40] - 65504) < 65504 * 2.0 ** -10 and (v[2, 0, :32] == 1.0).all()
    assert v[3, 0, 7] == -65504
    assert (v[4] == 65504).all()


def test_page_bytes():
    for d in HEAD_SIZES:
        for bs in (16, 32, 1024):
            assert KV4.kv4_page_bytes(d, bs) == bs * K4.groups(d) * 20
    lib = _lib.backend()
    for d, bs, want in ((40, 16, NXT_ATTN_E_UNSUPPORTED), (128, 8, NXT_ATTN_E_UNSUPPORTED),
                        (128, 24, NXT_ATTN_E_UNSUPPORTED), (128, 2048, NXT_ATTN_E_UNSUPPORTED),
                        (128, 0, NXT_ATTN_E_INVALID), (128, -16, NXT_ATTN_E_INVALID),
                        (0, 16, NXT_ATTN_E_UNSUPPORTED)):
        assert lib.nxt_paged_kv4_page_bytes(d, bs) == want
        assert lib.nxt_attn_last_status() == want and lib.nxt_attn_last_error()


P = 1 << 20  # stands for a device address: a refused call never reads it
PAGE = 1280  # head_size 128, block_size 16

APPEND = dict(kc=P, vc=P, key=P, value=P, bt=P, pos=P, n=2, kvh=8, d=128, mb=4, bs=16,
              bstride=8 * PAGE, hstride=PAGE, dtype=NXT_KV_FP16)
SLOTS = dict(kc=P, vc=P, key=P, value=P, slots=P, n=2, kvh=8, d=128, bs=16, bstride=8 * PAGE,
             hstride=PAGE, dtype=NXT_KV_FP16)
COPY = dict(kc=P, vc=P, src=P, dst=P, n=2, kvh=8, d=128, bs=16, bstride=8 * PAGE, hstride=PAGE)
ATTN = dict(out=P, q=P, kc=P, vc=P, bt=P, lens=P, n=2, h=32, d=128, kvh=8, scale=0.1, mb=4, bs=16,
            bstride=8 * PAGE, hstride=PAGE, dtype=NXT_KV_FP16)
CALLS = {"nxt_paged_kv4_append": APPEND, "nxt_paged_kv4_write_slots": SLOTS,
         "nxt_paged_kv4_read_slots": SLOTS, "nxt_paged_kv4_copy_slots": COPY,
         "nxt_paged_attention_kv4": ATTN}
INV, UNS = NXT_ATTN_E_INVALID, NXT_ATTN_E_UNSUPPORTED
REFUSALS = [("n", -1, INV), ("kvh", 0, INV), ("kvh", -8, INV), ("d", 40, UNS), ("d", 0, UNS),
            ("bs", 8, UNS), ("bs", 48, UNS), ("bs", 2048, UNS), ("bs", 0, INV),
            ("bstride", PAGE - 16, INV), ("hstride", PAGE - 16, INV), ("hstride", -PAGE, INV),
            ("bstride", -8 * PAGE, INV), ("bstride", 8 * PAGE + 8, UNS), ("hstride", PAGE + 4, UNS),
            ("dtype", 0, UNS), ("dtype", 4, UNS), ("mb", 0, INV), ("mb", -1, INV),
            ("mb", 1 << 25, UNS), ("kc", 0, INV), ("vc", 0, INV), ("key", 0, INV),
            ("value", 0, INV), ("bt", 0, INV), ("pos", 0, INV), ("slots", 0, INV), ("src", 0, INV),
            ("dst", 0, INV), ("out", 0, INV), ("q", 0, INV), ("lens", 0, INV), ("kc", P + 8, UNS),
            ("vc", P + 4, UNS), ("key", P + 2, UNS), ("value", P + 8, UNS), ("out", P + 8, UNS),
            ("q", P + 4, UNS), ("bt", P + 2, INV), ("pos", P + 1, INV), ("slots", P + 2, INV),
            ("src", P + 3, INV), ("dst", P + 1, INV), ("lens", P + 2, INV), ("h", 31, INV),
            ("h", 0, INV), ("h", 8 * 65, UNS), ("scale", float("inf"), INV),
            ("scale", float("nan"), INV), ("kvh", 1 << 25, UNS)]


def _call(name, args):
    a = [ctypes.c_float(v) if k == "scale" else v for k, v in args.items()]
    if name == "nxt_paged_attention_kv4":
        pass
    return getattr(_lib.backend(), name)(*a, None)


@pytest.mark.parametrize("name", sorted(CALLS))
def test_c_entry_points_refuse(name):
    base = CALLS[name]
    tried = 0
    for key, value, want in REFUSALS:
        if key not in base or (key == "kvh" and value > 1000 and "h" in base):
            continue
        args = dict(base, **{key: value})
        assert _call(name, args) == want, (name, key, value, _lib.backend().nxt_attn_last_error())
        assert _lib.backend().nxt_attn_last_status() == want
        tried += 1
    assert tried > 15


@pytest.mark.parametrize("name", sorted(CALLS))
def test_no_tokens_is_no_work(name):
    null = {k: 0 for k in CALLS[name] if k in ("out", "q", "kc", "vc", "bt", "lens", "key", "value",
                                               "pos", "slots", "src", "dst")}
    assert _call(name, dict(CALLS[name], n=0, **null)) == NXT_ATTN_OK
    # but a wrong shape is refused all the same
    assert _call(name, dict(CALLS[name], n=0, d=40, **null)) == UNS


@pytest.mark.parametrize("dtype", [NXT_KV_FP16, NXT_KV_BF16, NXT_KV_FP32])
def test_dtypes_are_taken(dtype):
    assert _call("nxt_paged_kv4_append", dict(APPEND, n=0, dtype=dtype)) == NXT_ATTN_OK
    assert _call("nxt_paged_attention_kv4", dict(ATTN, n=0, dtype=dtype)) == NXT_ATTN_OK


def test_python_calls_refuse_cpu_tensors():
    kc = torch.zeros((4, 2, KV4.kv4_page_bytes(64, 16)), dtype=torch.uint8)
    row = torch.zeros((3, 2, 64), dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        KV4.paged_kv4_append(kc, kc, row, row, slot_mapping=slots)
    with pytest.raises(ValueError):
        KV4.paged_kv4_read(row, row, kc, kc, slots)
    with pytest.raises(ValueError):
        KV4.paged_kv4_copy_slots(kc, kc, slots, slots, head_size=64)
    with pytest.raises(ValueError):
        KV4.paged_attention_kv4(row, row, kc, kc, slots[:, None], slots, num_kv_heads=2, scale=1.0)
