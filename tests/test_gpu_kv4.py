"""The 4-bit cache operators on the GPU: rows to the bit, attention against 64
bits within tests/kv4_cases.attention_bound."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import kv4_cases as C
from oracle import kv4_oracle as K4
from xllms_amd import kv4_cache as KV4
from xllms_amd import paged_attention as PA

pytestmark = pytest.mark.gpu


def _dev(x):
    return torch.as_tensor(x).to("cuda")


def _cache(pool, kvh, d, bs, fill=0xAA):
    return tuple(torch.full((pool, kvh, KV4.kv4_page_bytes(d, bs)), fill, dtype=torch.uint8,
                            device="cuda") for _ in "kv")


def _write(kc, vc, k, v, slots):
    KV4.paged_kv4_append(kc, vc, _dev(k), _dev(v), slot_mapping=_dev(slots))


def _same(got, want):
    """Equal to the bit, any NaN equal to any NaN."""
    g, w = got.cpu(), want.cpu()
    assert g.dtype == w.dtype
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    assert torch.equal(torch.nan_to_num(g.double()), torch.nan_to_num(w.double()))


def _stored(rows, dtype):
    """What read_slots returns: fp32 values rounded to dtype."""
    a, lo = K4.split(*K4.quantise(C.np32(rows)))
    return torch.from_numpy((a + lo).astype(np.float32)).to(C.DTYPES[dtype])


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("d", [32, 64, 80, 96, 112, 128, 192, 256])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_written_rows_read_back(cuda, d, dtype):
    n, kvh, bs = 77, 3, 32
    k, v = C.rows(n, kvh, d, dtype, d), C.rows(n, kvh, d, dtype, d + 1)
    k[3] = 0.25                     # constant rows
    k[5] *= 1e-6                    # steps and lows below the normal fp16 range
    v[7] *= 3e4                     # past the fp16 range where the type holds it
    v[9, 1, 2] = float("nan")
    k[11, 2, d - 1] = float("inf")
    v[11, 0, 0] = float("-inf")
    rng = np.random.default_rng(d)
    slots = rng.permutation(6 * bs)[:n].astype(np.int32)
    slots[13] = -1                  # not written, not read
    kc, vc = _cache(6, kvh, d, bs)
    _write(kc, vc, k, v, slots)
    for out in ("fp16", "bf16", "fp32"):
        ko = torch.full((n, kvh, d), 7.0, dtype=C.DTYPES[out], device="cuda")
        vo = ko.clone()
        KV4.paged_kv4_read(ko, vo, kc, vc, _dev(slots))
        wk, wv = _stored(k, out), _stored(v, out)
        wk[13] = wv[13] = 7.0
        _same(ko, wk)
        _same(vo, wv)


def test_step_is_rounded_twice(cuda):
    """Ranges whose fifteenth, rounded to fp32 on its way to fp16, is not the fp16
    number nearest to it."""
    g = torch.Generator().manual_seed(15)
    x = torch.randn((400000, 32), generator=g)
    span = (x.max(1).values - x.min(1).values).numpy()
    exact = span.astype(np.float64) * np.float64(np.float32(1.0 / 15.0))
    pick = exact.astype(np.float16) != exact.astype(np.float32).astype(np.float16)
    assert pick.sum() >= 5
    k = x[torch.from_numpy(pick)][:, None].contiguous()
    n = k.shape[0]
    kc, vc = _cache(-(-n // 16), 1, 32, 16)
    slots = np.arange(n, dtype=np.int32)
    _write(kc, vc, k, k, slots)
    ko, vo = (torch.empty((n, 1, 32), device="cuda") for _ in "kv")
    KV4.paged_kv4_read(ko, vo, kc, vc, _dev(slots))
    _same(ko, _stored(k, "fp32"))
    _same(vo, _stored(k, "fp32"))


@pytest.mark.parametrize("bs", [16, 64, 1024])
def test_append_by_tables(cuda, bs):
    """Tokens at the edges of pages and tiles; skipped positions; other slots
    and other pages keep their bytes."""
    kvh, d, dtype = 2, 96, "bf16"
    pos = np.array([0, 1, 15, 16, bs - 1, bs, 2 * bs - 1, -1, 2 * bs, 5, 7], dtype=np.int32)
    bt = np.arange(2 * len(pos), dtype=np.int32).reshape(-1, 2)[:, ::-1].copy()
    bt[9, 0] = -1                   # a page that is not there
    k, v = C.rows(len(pos), kvh, d, dtype, 1), C.rows(len(pos), kvh, d, dtype, 2)
    kc, vc = _cache(bt.size, kvh, d, bs)
    KV4.paged_kv4_append(kc, vc, _dev(k), _dev(v), block_tables=_dev(bt), positions=_dev(pos))
    done = [s for s in range(len(pos)) if 0 <= pos[s] < 2 * bs and bt[s, pos[s] // bs] >= 0]
    assert len(done) == len(pos) - 3
    slots = np.array([bt[s, pos[s] // bs] * bs + pos[s] % bs for s in done], dtype=np.int32)
    want_k, want_v = _cache(bt.size, kvh, d, bs)
    _write(want_k, want_v, k[done], v[done], slots)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    ko, vo = (torch.empty((len(done), kvh, d), dtype=C.DTYPES[dtype], device="cuda") for _ in "kv")
    KV4.paged_kv4_read(ko, vo, kc, vc, _dev(slots))
    _same(ko, _stored(k[done], dtype))
    _same(vo, _stored(v[done], dtype))
    # a row is 20 bytes a group of K and of V: nothing else changed
    for c in (kc, vc):
        assert int((c != 0xAA).sum()) <= len(done) * kvh * K4.groups(d) * 20


def test_one_token_and_one_by_one(cuda):
    """A prompt written at once, and token by token: the same bytes."""
    n, kvh, d, bs = 37, 2, 80, 16
    k, v = C.rows(n, kvh, d, "fp16", 3), C.rows(n, kvh, d, "fp16", 4)
    slots = np.arange(n, dtype=np.int32) + 5
    a, b = _cache(3, kvh, d, bs), _cache(3, kvh, d, bs)
    _write(*a, k, v, slots)
    for i in range(n):
        _write(*b, k[i:i + 1], v[i:i + 1], slots[i:i + 1])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_strided_caches(cuda):
    """Pages inside a larger buffer, and a head-major pool."""
    n, kvh, d, bs, pool = 40, 3, 64, 16, 4
    page = KV4.kv4_page_bytes(d, bs)
    k, v = C.rows(n, kvh, d, "fp32", 5), C.rows(n, kvh, d, "fp32", 6)
    slots = np.random.default_rng(0).permutation(pool * bs)[:n].astype(np.int32)
    plain = _cache(pool, kvh, d, bs)
    _write(*plain, k, v, slots)
    wide = [torch.full((pool, kvh + 2, page + 48), 0xAA, dtype=torch.uint8, device="cuda") for _ in "kv"]
    major = [torch.full((kvh, pool, page), 0xAA, dtype=torch.uint8, device="cuda") for _ in "kv"]
    for views in ([w[:, 1:1 + kvh, 16:16 + page] for w in wide], [m.transpose(0, 1) for m in major]):
        _write(*views, k, v, slots)
        assert torch.equal(views[0].contiguous(), plain[0])
        assert torch.equal(views[1].contiguous(), plain[1])
        ko, vo = (torch.empty((n, kvh, d), device="cuda") for _ in "kv")
        KV4.paged_kv4_read(ko, vo, *views, _dev(slots))
        _same(ko, _stored(k, "fp32"))
        _same(vo, _stored(v, "fp32"))
    for w in wide:  # around the pages
        w[:, 1:1 + kvh, 16:16 + page] = 0xAA
        assert bool((w == 0xAA).all())


@pytest.mark.parametrize("d,bs", [(128, 16), (80, 64), (256, 32)])
def test_copy_slots(cuda, d, bs):
    kvh, pool = 2, 5
    n = pool * bs
    k, v = C.rows(n, kvh, d, "bf16", 7), C.rows(n, kvh, d, "bf16", 8)
    kc, vc = _cache(pool, kvh, d, bs)
    _write(kc, vc, k, v, np.arange(n, dtype=np.int32))
    perm = np.random.default_rng(1).permutation(n)
    src, dst = perm[:n // 3].astype(np.int32), perm[n // 3:2 * (n // 3)].astype(np.int32)
    src[4], dst[9] = -1, -1
    KV4.paged_kv4_copy_slots(kc, vc, _dev(src), _dev(dst), head_size=d)
    ok = (src >= 0) & (dst >= 0)
    k[dst[ok]], v[dst[ok]] = k[src[ok]], v[src[ok]]
    want = _cache(pool, kvh, d, bs)
    _write(*want, k, v, np.arange(n, dtype=np.int32))
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_pages_past_4_gib(cuda):
    """Offsets that need more than 32 bits: rows, copy and attention in the
    last pages of a cache of over 4 GiB."""
    kvh, d, bs = 8, 128, 16
    page = kvh * KV4.kv4_page_bytes(d, bs)
    pool = (1 << 32) // page + 100
    kc, vc = (torch.empty((pool, kvh, page // kvh), dtype=torch.uint8, device="cuda") for _ in "kv")
    lens = [45]
    bt = np.array([[pool - 1, pool - 40, pool - 7]], dtype=np.int32)
    k, v = C.rows(45, kvh, d, "fp16", 9), C.rows(45, kvh, d, "fp16", 10)
    slots = C.slots_for(bt, lens, bs)
    _write(kc, vc, k, v, slots)
    ko, vo = (torch.empty((45, kvh, d), dtype=torch.float16, device="cuda") for _ in "kv")
    KV4.paged_kv4_read(ko, vo, kc, vc, _dev(slots))
    _same(ko, _stored(k, "fp16"))
    _same(vo, _stored(v, "fp16"))
    q = C.rows(1, 32, d, "fp16", 11)
    _check(_attend(q, kc, vc, bt, lens, kvh), "fp16", C.reference(q, k, v, lens, C.scale_of(d), kvh))
    moved = np.array([[pool - 2, pool - 41, pool - 8]], dtype=np.int32)
    KV4.paged_kv4_copy_slots(kc, vc, _dev(slots), _dev(C.slots_for(moved, lens, bs)), head_size=d)
    assert torch.equal(_attend(q, kc, vc, moved, lens, kvh), _attend(q, kc, vc, bt, lens, kvh))


# ------------------------------------------------------------- attention
def _attend(q, kc, vc, bt, lens, kvh, scale=None, **kw):
    qd = _dev(q)
    out = torch.full_like(qd, 7.0)
    KV4.paged_attention_kv4(out, qd, kc, vc, _dev(np.asarray(bt)), _dev(np.asarray(lens, np.int32)),
                            num_kv_heads=kvh, scale=C.scale_of(q.shape[-1]) if scale is None else scale,
                            **kw)
    return out


def _check(got, dtype, ref):
    got = C.np64(got)
    assert np.isfinite(got).all()
    err, bound = np.abs(got - ref[0]), C.attention_bound(dtype, *ref)
    worst = (err / bound).max()
    print(f"error / bound {worst:.3f}")
    assert worst <= 1.0, (worst, np.unravel_index((err / bound).argmax(), err.shape))


def _batch(dtype, h, kvh, d, bs, lens, seed=0):
    """(q, k rows, v rows, caches, block tables) of a batch in a shuffled pool
    whose other slots hold bytes of NaN lows and steps."""
    n = sum(lens)
    q = C.rows(len(lens), h, d, dtype, seed)
    k, v = C.rows(n, kvh, d, dtype, seed + 1), C.rows(n, kvh, d, dtype, seed + 2)
    bt, pool = C.tables_for(lens, bs, seed)
    kc, vc = _cache(pool, kvh, d, bs, fill=0xFF)
    _write(kc, vc, k, v, C.slots_for(bt, lens, bs))
    return q, k, v, kc, vc, bt


RAGGED = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 200, 1000, 0, 129]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("h,kvh,d,bs", [(8, 2, 128, 16), (4, 4, 64, 16), (6, 2, 80, 32),
                                        (2, 1, 32, 64), (5, 1, 96, 16), (7, 1, 112, 16),
                                        (6, 2, 192, 128), (4, 2, 256, 16)])
def test_ragged_batch(cuda, dtype, h, kvh, d, bs):
    q, k, v, kc, vc, bt = _batch(dtype, h, kvh, d, bs, RAGGED)
    _check(_attend(q, kc, vc, bt, RAGGED, kvh), dtype, C.reference(q, k, v, RAGGED, C.scale_of(d), kvh))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("group", [1, 3, 8, 15, 16, 17, 24, 32, 33, 48, 49, 64])
def test_groups_of_query_heads(cuda, dtype, group):
    lens = [50, 333, 7]
    q, k, v, kc, vc, bt = _batch(dtype, 2 * group, 2, 128, 16, lens, seed=group)
    _check(_attend(q, kc, vc, bt, lens, 2), dtype, C.reference(q, k, v, lens, C.scale_of(128), 2))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("h,kvh,d,bs", [(32, 2, 128, 16), (18, 2, 64, 16), (16, 1, 32, 16),
                                        (12, 1, 80, 32), (44, 4, 112, 16), (40, 1, 192, 16)])
def test_larger_groups_with_cut_segments(cuda, dtype, h, kvh, d, bs):
    """Groups of 9 to 40 heads: segments over many workgroups, inside one, and
    several in one wavefront's range (2400 sequences of 1 to 160 tokens)."""
    lens = [3000, 900] + RAGGED + [1 + (i * 37) % 160 for i in range(2400)] + [2100]
    q, k, v, kc, vc, bt = _batch(dtype, h, kvh, d, bs, lens, seed=h)
    out = _attend(q, kc, vc, bt, lens, kvh)
    pick = list(range(0, len(lens), 43)) + [1, len(lens) - 1]
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
    ref = C.reference(q[pick], k, v, [lens[i] for i in pick], C.scale_of(d), kvh, starts[pick])
    _check(out[pick], dtype, ref)
    for _ in range(5):
        assert torch.equal(_attend(q, kc, vc, bt, lens, kvh), out)


def test_larger_groups_with_nan_and_missing_pages(cuda):
    """A NaN query, NaN values and pages that are not there stay with their heads
    and sequences where pieces are joined."""
    kvh, d, bs = 2, 128, 16
    lens = [500, 40, 100] + [1 + (i * 29) % 150 for i in range(2200)]
    q, k, v, kc, vc, bt = _batch("fp16", 16 * kvh, kvh, d, bs, lens, seed=1)
    want = _attend(q, kc, vc, bt, lens, kvh)
    q2, cut = q.clone(), bt.copy()
    q2[0, 5, 7] = float("nan")
    q2[900, 20] = float("inf")
    cut[1, :] = -1
    cut[2, 3:] = -1
    v2 = v[:lens[0]].clone()
    v2[480, 1, 100] = float("nan")
    _write(kc, vc, k[:lens[0]], v2, C.slots_for(bt[:1], lens[:1], bs))
    out = _attend(q2, kc, vc, cut, lens, kvh)
    assert torch.isnan(out[0, 5]).all() and torch.isnan(out[900, 20]).all()
    assert torch.isnan(out[0, 16:, 96:]).all()
    assert bool((out[1] == 0).all())
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
    ref = C.reference(q[2:3], k, v, [3 * bs], C.scale_of(d), kvh, starts[2:3])
    _check(out[2:3], "fp16", ref)
    # (the step of a NaN row lowers the weights' scale for its kv head: other bits)
    ref = C.reference(q[:1], k, v, lens[:1], C.scale_of(d), kvh, starts[:1])
    _check(out[:1, 16:, :96], "fp16", [r[:, 16:, :96] if r.ndim == 3 else r[:, 16:] for r in ref])
    same = torch.ones_like(out, dtype=torch.bool)
    same[0, 5], same[900, 20], same[1], same[2], same[0, 16:] = (False,) * 5
    assert torch.equal(out[same], want[same])


@pytest.mark.parametrize("dtype,d", [("fp16", 128), ("bf16", 256), ("fp32", 64), ("fp32", 256)])
def test_one_long_sequence(cuda, dtype, d):
    """Split over the whole GPU, with keys that make sharp peaks."""
    lens = [9001]
    q, k, v, kc, vc, bt = _batch(dtype, 4, 1, d, 16, lens, seed=5)
    k[::97] *= 4.0
    _write(kc, vc, k, v, C.slots_for(bt, lens, 16))
    _check(_attend(q, kc, vc, bt, lens, 1), dtype, C.reference(q, k, v, lens, C.scale_of(d), 1))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("h,d", [(4, 128), (16, 128), (32, 64), (4, 80), (16, 192), (8, 256)])
def test_long_ranges(cuda, dtype, h, d):
    """Ranges of dozens of tiles, that end anywhere, in every form of the kernel."""
    n, L = 1500, 2047
    q = C.rows(n, h, d, dtype, 1)
    k, v = C.rows(L, 1, d, dtype, 2), C.rows(L, 1, d, dtype, 3)
    bt, pool = C.tables_for([L], 16, 0)
    kc, vc = _cache(pool, 1, d, 16, fill=0xFF)
    _write(kc, vc, k, v, C.slots_for(bt, [L], 16))
    lens = [L - 3 * (i % 50) for i in range(n)]
    out = _attend(q, kc, vc, np.repeat(bt, n, 0), lens, 1)
    pick = [0, 49, 700, n - 1]
    ref = C.reference(q[pick], k, v, [lens[i] for i in pick], C.scale_of(d), 1, [0] * len(pick))
    _check(out[pick], dtype, ref)


def test_many_sequences(cuda):
    """More sequences than one launch takes."""
    lens = [1 + (i * 7) % 40 for i in range(8200)]
    lens[5] = lens[8195] = 0
    d, kvh = 32, 1
    q, k, v, kc, vc, bt = _batch("fp16", 2, kvh, d, 16, lens, seed=2)
    out = _attend(q, kc, vc, bt, lens, kvh)
    pick = list(range(0, 60)) + list(range(8150, 8200))
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
    ref = C.reference(q[pick], k, v, [lens[i] for i in pick], C.scale_of(d), kvh, starts[pick])
    _check(out[pick], "fp16", ref)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("size_v", [1e-4, 1.0, 40.0, 2000.0])
def test_sizes_of_values(cuda, dtype, size_v):
    """Steps of V from below the normal fp16 range to far above 1, in one
    sequence, and queries from tiny to large."""
    lens = [90, 300]
    q, k, v, kc, vc, bt = _batch(dtype, 8, 2, 64, 16, lens, seed=4)
    q[0] *= 1e-3
    q[1] *= 6.0
    v = (v.float() * size_v).to(v.dtype)
    v[40:60] *= 5.0
    _write(kc, vc, k, v, C.slots_for(bt, lens, 16))
    _check(_attend(q, kc, vc, bt, lens, 2), dtype, C.reference(q, k, v, lens, C.scale_of(64), 2))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("exp", [-60, 60])
def test_queries_far_from_one(cuda, dtype, exp):
    """Query magnitudes outside fp16, brought back by the scale."""
    lens = [70]
    q, k, v, kc, vc, bt = _batch(dtype, 4, 1, 128, 16, lens, seed=6)
    q = (q.double() * 2.0 ** exp).to(q.dtype)
    scale = C.scale_of(128) * 2.0 ** -exp
    _check(_attend(q, kc, vc, bt, lens, 1, scale=scale), dtype, C.reference(q, k, v, lens, scale, 1))


@pytest.mark.parametrize("h,kvh,d", [(12, 12, 64), (8, 2, 128), (32, 2, 128), (24, 1, 96)])
def test_fp32_keeps_its_bits(cuda, h, kvh, d):
    """Root mean square error of fp32 outputs.  Scores of parts below 32 (log2
    units) take about five roundings of at most 2^-20 each, 2^-20.8 rms, which
    move the weights by ln 2 of that, independently: sqrt(5) * 2^-21.3 = 2^-20.2
    of the output; and the sums' own, 2^-26 of the sizes, which are below 64
    outputs here: 2^-20.  Together 2^-19.1."""
    lens = [1000, 517, 1000, 64]
    g = torch.Generator().manual_seed(d + h)
    q = 0.25 * torch.randn((len(lens), h, d), generator=g)
    k, v = (torch.randn((sum(lens), kvh, d), generator=g) for _ in "kv")
    bt, pool = C.tables_for(lens, 16, 0)
    kc, vc = _cache(pool, kvh, d, 16, fill=0xFF)
    _write(kc, vc, k, v, C.slots_for(bt, lens, 16))
    ref = C.reference(q, k, v, lens, C.scale_of(d), kvh)
    assert ref[2].max() * np.log2(np.e) < 32
    err = C.np64(_attend(q, kc, vc, bt, lens, kvh)) - ref[0]
    rel = np.sqrt((err ** 2).mean() / (ref[0] ** 2).mean())
    print(f"rms {rel:.2e}")
    assert rel < 2.0 ** -19


def test_long_ranges_do_not_drift(cuda):
    """8192 tokens times 2000 sequences of one set of pages: whole sequences in a
    wavefront's range, nearly equal weights, outputs far below the values."""
    n, d = 2000, 32
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((8192, 1, d), generator=g) for _ in "kv")
    bt, pool = C.tables_for([8192], 16, 0)
    for dtype, most in (("fp32", 1e-4), ("fp16", 2.0 ** -12 + 1e-4)):
        q = (0.1 * torch.randn((n, 2, d), generator=g)).to(C.DTYPES[dtype])
        kd, vd = k.to(C.DTYPES[dtype]), v.to(C.DTYPES[dtype])
        kc, vc = _cache(pool, 1, d, 16)
        _write(kc, vc, kd, vd, C.slots_for(bt, [8192], 16))
        out = _attend(q, kc, vc, np.repeat(bt, n, 0), [8192] * n, 1)
        ref = C.reference(q[:3], kd, vd, [8192] * 3, C.scale_of(d), 1, [0, 0, 0])[0]
        rel = np.sqrt(((C.np64(out[:3]) - ref) ** 2).mean() / (ref ** 2).mean())
        print(f"{dtype} rms {rel:.2e}")
        assert rel < most


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_query_and_scale_far_apart(cuda, dtype):
    """A scale whose product with a constant alone would pass fp32's range."""
    lens = [70]
    q, k, v, kc, vc, bt = _batch(dtype, 4, 1, 128, 16, lens, seed=6)
    q = (q.double() * 2.0 ** -112).to(q.dtype)
    scale = C.scale_of(128) * 2.0 ** 112
    _check(_attend(q, kc, vc, bt, lens, 1, scale=scale), dtype, C.reference(q, k, v, lens, scale, 1))


def test_queries_of_zero(cuda):
    lens = [33]
    q, k, v, kc, vc, bt = _batch("fp16", 4, 2, 64, 16, lens)
    q.zero_()
    _check(_attend(q, kc, vc, bt, lens, 2), "fp16", C.reference(q, k, v, lens, C.scale_of(64), 2))


def test_one_token_is_its_value(cuda):
    """A weight of 1 is exact, so a context of one token is what is stored."""
    lens = [1, 1, 1]
    for dtype in ("fp16", "bf16", "fp32"):
        q, k, v, kc, vc, bt = _batch(dtype, 6, 2, 128, 16, lens, seed=8)
        out = _attend(q, kc, vc, bt, lens, 2).reshape(3, 2, 3, 128)
        _same(out, _stored(v, dtype)[:, :, None].expand(3, 2, 3, 128))


@pytest.mark.parametrize("bs", [16, 64])
def test_missing_pages_contribute_nothing(cuda, bs):
    """Negative page ids: whole sequences, single pages, and one between
    others; the rest of the batch is untouched by them."""
    lens = [3 * bs + 5, 2 * bs, bs - 3]
    q, k, v, kc, vc, bt = _batch("fp16", 8, 2, 128, bs, lens, seed=9)
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
    cut = bt.copy()
    cut[0, 1] = -1
    cut[2, :] = -5
    out = _attend(q, kc, vc, cut, lens, 2)
    keep = np.r_[0:bs, 2 * bs:lens[0]]
    r0 = C.reference(q[:1], k[keep], v[keep], [len(keep)], C.scale_of(128), 2)
    _check(out[:1], "fp16", r0)
    _check(out[1:2], "fp16", C.reference(q[1:2], k, v, [lens[1]], C.scale_of(128), 2, starts[1:2]))
    assert bool((out[2] == 0).all())


def test_nan_rows_reach_their_heads_only(cuda):
    lens = [100]
    q, k, v, kc, vc, bt = _batch("fp16", 4, 2, 64, 16, lens, seed=10)
    v[50, 1, 40] = float("nan")
    _write(kc, vc, k, v, C.slots_for(bt, lens, 16))
    out = _attend(q, kc, vc, bt, lens, 2)[0]
    assert torch.isnan(out[2:, 32:]).all()
    assert torch.isfinite(out[:2]).all()
    k[20, 0, 3] = float("nan")
    _write(kc, vc, k, v, C.slots_for(bt, lens, 16))
    out = _attend(q, kc, vc, bt, lens, 2)[0]
    assert torch.isnan(out[:2]).all()


def test_lengths_past_the_table_are_clamped(cuda):
    lens = [48, 20]
    q, k, v, kc, vc, bt = _batch("bf16", 8, 2, 128, 16, lens, seed=11)
    assert bt.shape[1] == 3
    want = _attend(q, kc, vc, bt, lens, 2)
    assert torch.equal(_attend(q, kc, vc, bt, [5000, 20], 2), want)
    assert bool((_attend(q, kc, vc, bt, [-3, 20], 2)[0] == 0).all())


def test_strided_cache_and_bits(cuda):
    """A head-major pool gives the same bits, and so does a second call."""
    lens = [500, 33, 260]
    q, k, v, kc, vc, bt = _batch("fp16", 32, 8, 128, 16, lens, seed=12)
    a = _attend(q, kc, vc, bt, lens, 8)
    assert torch.equal(a, _attend(q, kc, vc, bt, lens, 8))
    km, vm = (c.transpose(0, 1).contiguous().transpose(0, 1) for c in (kc, vc))
    assert torch.equal(a, _attend(q, km, vm, bt, lens, 8))


def test_decode_loop(cuda):
    """Prompts written by slots, then steps of append and attention, a copy of
    a page to a second sequence, and the read back of it all."""
    kvh, h, d, bs, steps = 2, 8, 128, 16, 40
    lens = [30, 1]
    bt = np.array([[3, 0, 6, 1, 8], [2, 7, 4, 9, 5]], dtype=np.int32)
    kc, vc = _cache(10, kvh, d, bs, fill=0xFF)
    hist = [[C.rows(n, kvh, d, "bf16", 20 + s), C.rows(n, kvh, d, "bf16", 30 + s)]
            for s, n in enumerate(lens)]
    for s in range(2):
        _write(kc, vc, *hist[s], C.slots_for(bt[s:s + 1], lens[s:s + 1], bs))
    dbt = _dev(bt)
    for i in range(steps):
        k, v = C.rows(2, kvh, d, "bf16", 100 + i), C.rows(2, kvh, d, "bf16", 200 + i)
        KV4.paged_kv4_append(kc, vc, _dev(k), _dev(v), block_tables=dbt,
                             positions=_dev(np.array(lens, np.int32)))
        for s in range(2):
            hist[s] = [torch.cat([hist[s][j], x[s:s + 1]]) for j, x in enumerate((k, v))]
        lens = [n + 1 for n in lens]
        if i % 13 == 0 or i == steps - 1:
            q = C.rows(2, h, d, "bf16", 300 + i)
            ref = C.reference(q, torch.cat([x[0] for x in hist]), torch.cat([x[1] for x in hist]),
                              lens, C.scale_of(d), kvh)
            _check(_attend(q, kc, vc, bt, lens, kvh), "bf16", ref)
    # sequence 1 forks from sequence 0: its first page becomes a copy
    src = _dev(bt[0, 0] * bs + np.arange(bs, dtype=np.int32))
    dst = _dev(bt[1, 0] * bs + np.arange(bs, dtype=np.int32))
    KV4.paged_kv4_copy_slots(kc, vc, src, dst, head_size=d)
    for j in range(2):
        hist[1][j][:bs] = hist[0][j][:bs]
    slots = C.slots_for(bt, lens, bs)
    ko, vo = (torch.empty((sum(lens), kvh, d), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    KV4.paged_kv4_read(ko, vo, kc, vc, _dev(slots))
    _same(ko, _stored(torch.cat([x[0] for x in hist]), "bf16"))
    _same(vo, _stored(torch.cat([x[1] for x in hist]), "bf16"))


# ------------------------------------------------- streams, graphs, refusals
def test_two_streams_at_once(cuda):
    sets = []
    for i in range(2):
        lens = [700 + 900 * i, 64, 3]
        sets.append((_batch("fp16", 32, 8, 128, 16, lens, seed=40 + i), lens))
    want = [_attend(b[0], *b[3:], lens, 8) for b, lens in sets]
    args = [(_dev(b[0]), b[3], b[4], _dev(b[5]), _dev(np.array(lens, np.int32))) for b, lens in sets]
    outs = [torch.zeros_like(w) for w in want]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, out, (q, kc, vc, bt, ln) in zip(streams, outs, args):
            with torch.cuda.stream(st):
                out.zero_()
                KV4.paged_attention_kv4(out, q, kc, vc, bt, ln, num_kv_heads=8, scale=C.scale_of(128))
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)


def test_captured_step_replays(cuda):
    """Append, attention and read back in one graph; lengths, positions, rows
    and queries change between replays, with eager calls in between."""
    kvh, h, d, bs = 2, 8, 128, 16
    lens = [600, 40, 0]
    q, k, v, kc, vc, bt = _batch("fp16", h, kvh, d, bs, lens, seed=50)
    bt, pool = C.tables_for([700, 100, 100], bs, 50)
    kc, vc = _cache(pool, kvh, d, bs, fill=0xFF)
    _write(kc, vc, k, v, C.slots_for(bt, lens, bs))
    dq, dbt = _dev(q), _dev(bt)
    nk, nv = (torch.empty((3, kvh, d), dtype=torch.float16, device="cuda") for _ in "kv")
    pos, ln, slots = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    out, ko, vo = torch.empty_like(dq), torch.empty_like(nk), torch.empty_like(nv)

    def step(o, a, b):
        KV4.paged_kv4_append(kc, vc, nk, nv, block_tables=dbt, positions=pos)
        KV4.paged_attention_kv4(o, dq, kc, vc, dbt, ln, num_kv_heads=kvh, scale=C.scale_of(d))
        KV4.paged_kv4_read(a, b, kc, vc, slots)

    def load(i):
        nk.copy_(C.rows(3, kvh, d, "fp16", 60 + i))
        nv.copy_(C.rows(3, kvh, d, "fp16", 70 + i))
        dq.copy_(C.rows(3, h, d, "fp16", 80 + i))
        at = np.array([n + i for n in lens], np.int32)
        pos.copy_(_dev(at))
        ln.copy_(_dev(at + 1))
        slots.copy_(_dev(np.array([bt[s, p // bs] * bs + p % bs for s, p in enumerate(at)], np.int32)))

    st = torch.cuda.Stream()
    load(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step(out, ko, vo)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        step(out, ko, vo)
    for i in range(6):
        load(i)
        for t in (out, ko, vo):
            t.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        e = [torch.empty_like(t) for t in (out, ko, vo)]
        step(*e)
        torch.cuda.synchronize()
        for got, want in zip((out, ko, vo), e):
            assert torch.equal(got, want)
        _same(ko, _stored(nk, "fp16"))


def test_refused_calls_leave_the_output(cuda):
    lens = [20]
    q, k, v, kc, vc, bt = _batch("fp16", 4, 2, 64, 16, lens)
    out = torch.full_like(_dev(q), 7.0)
    ln = _dev(np.array(lens, np.int32))
    with pytest.raises(PA.PagedAttentionError):
        KV4.paged_attention_kv4(out, _dev(q), kc, vc, _dev(bt), ln, num_kv_heads=2,
                                scale=float("nan"))
    for bad in (dict(num_kv_heads=1), dict(num_kv_heads=4), dict(num_kv_heads=2, block_size=32)):
        with pytest.raises(ValueError):
            KV4.paged_attention_kv4(out, _dev(q), kc, vc, _dev(bt), ln, scale=1.0, **bad)
    with pytest.raises(ValueError):
        KV4.paged_attention_kv4(out, _dev(q), kc, vc, _dev(bt).long(), ln, num_kv_heads=2, scale=1.0)
    with pytest.raises(ValueError):
        KV4.paged_attention_kv4(out, _dev(q), kc, vc, _dev(bt), ln.repeat(2), num_kv_heads=2, scale=1.0)
    row = torch.zeros((2, 2, 64), dtype=torch.float16, device="cuda")
    slot = torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: KV4.paged_kv4_append(kc, vc, row, row),
                 lambda: KV4.paged_kv4_append(kc, vc, row, row.float(), slot_mapping=slot),
                 lambda: KV4.paged_kv4_append(kc, vc, row[:, :1], row[:, :1], slot_mapping=slot),
                 lambda: KV4.paged_kv4_append(kc.half(), vc, row, row, slot_mapping=slot),
                 lambda: KV4.paged_kv4_read(row, row, kc, vc, slot[:1]),
                 lambda: KV4.paged_kv4_read(row, row, kc, vc, slot.long())):
        with pytest.raises(ValueError):
            call()
    assert bool((out == 7.0).all())


def test_more_refusals(cuda):
    q, k, v, kc, vc, bt = _batch("fp16", 4, 2, 64, 16, [20])
    row = torch.zeros((2, 2, 64), dtype=torch.float16, device="cuda")
    slot = torch.zeros(2, dtype=torch.int32, device="cuda")
    before = kc.clone()
    wide = torch.empty((2, (1 << 31) // KV4.kv4_page_bytes(64, 16) + 1, kc.shape[2]), dtype=torch.uint8,
                       device="cuda").transpose(0, 1)  # a head's pages past 2 GiB
    for call in (lambda: KV4.paged_kv4_append(wide, wide, row, row, slot_mapping=slot),
                 lambda: KV4.paged_kv4_append(kc, vc, row, row, slot_mapping=slot[:, None]),
                 lambda: KV4.paged_kv4_append(kc, vc, row, row, block_tables=slot, positions=slot),
                 lambda: KV4.paged_kv4_append(kc, vc, row[..., :0], row[..., :0], slot_mapping=slot),
                 lambda: KV4.paged_kv4_append(kc, vc, row.cpu(), row.cpu(), slot_mapping=slot),
                 lambda: KV4.paged_kv4_append(kc, vc, row, row, slot_mapping=slot.cpu()),
                 lambda: KV4.paged_kv4_append(kc.cpu(), vc.cpu(), row, row, slot_mapping=slot),
                 lambda: KV4.paged_kv4_copy_slots(kc, vc, slot, slot[:1], head_size=64),
                 lambda: KV4.paged_kv4_copy_slots(kc, vc, slot, slot, head_size=128, block_size=16),
                 lambda: KV4.paged_attention_kv4(row, row, kc, vc, slot, slot, num_kv_heads=2, scale=1.0)):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(kc, before)


def test_no_rows_from_python(cuda):
    kc, vc = _cache(2, 2, 64, 16)
    before = kc.clone()
    row = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    table = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    KV4.paged_kv4_append(kc, vc, row, row, slot_mapping=none)
    KV4.paged_kv4_append(kc, vc, row, row, block_tables=table, positions=none)
    KV4.paged_kv4_read(row, row, kc, vc, none)
    KV4.paged_kv4_copy_slots(kc, vc, none, none, head_size=64)
    KV4.paged_attention_kv4(row, row, kc, vc, table, none, num_kv_heads=2, scale=1.0)
    torch.cuda.synchronize()
    assert torch.equal(kc, before)


def test_repeated_calls_give_the_same_bits(cuda):
    """Many short sequences with partly filled tiles and missing pages: nothing
    depends on when a fetch comes back."""
    lens = [1 + (i * 7) % 90 for i in range(4000)]
    for d, kvh in ((32, 1), (128, 2)):
        q, k, v, kc, vc, bt = _batch("fp16", 2 * kvh, kvh, d, 16, lens, seed=3)
        bt[::5, 0] = -1
        want = _attend(q, kc, vc, bt, lens, kvh)
        for _ in range(15):
            assert torch.equal(_attend(q, kc, vc, bt, lens, kvh), want)
