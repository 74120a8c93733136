"""Python host mirror of the 4-bit K/V cache operators (torch tensors in).

Thin ctypes layer over libxllm_hip_backend.so, beside paged_attention.py: the
same decode attention, append, slot writes and slot copies over a paged cache
that holds K and V in 4 bits a channel, and the read back of its rows.  Every
call goes to the gfx950 kernels; there is no CPU path here.

Layouts:
  query / out   [num_seqs, num_heads, head_size]      fp16, bf16 or fp32
  key / value   [num_tokens, num_kv_heads, head_size] fp16, bf16 or fp32
  key_cache / value_cache  uint8 [num_blocks, num_kv_heads, page_bytes] (kv4_cache_empty);
                the strides of its first two dimensions are taken from the tensor
  block_tables  int32 [num_seqs, max_num_blocks_per_seq]
  seq_lens, positions, slot_mapping  int32

The format: groups of 32 channels of a row, value = low + step * code with low
and step in fp16 and a code of 0..15 (include/xllm_hip_operator_api.h has the
arithmetic).
"""
from __future__ import annotations

import ctypes

from . import _lib
from .paged_attention import (NXT_ATTN_OK, PagedAttentionError, _ptr, _stream_handle,
                              kv_dtype_of)

GROUP = 32  # channels that share a range
TILE = 16   # tokens of a tile: the smallest block_size


def _page_bytes(head_size: int, block_size: int) -> int:
    groups = (head_size + GROUP - 1) // GROUP
    return block_size * groups * (GROUP // 2 + 4)


def _raise(lib, status: int, check: bool) -> int:
    if check and status != NXT_ATTN_OK:
        raise PagedAttentionError(status, lib.nxt_attn_last_error().decode())
    return status


def kv4_page_bytes(head_size: int, block_size: int) -> int:
    """Bytes of one page of one kv head, of K and as many of V."""
    lib = _lib.backend()
    n = lib.nxt_paged_kv4_page_bytes(head_size, block_size)
    if n < 0:
        raise PagedAttentionError(n, lib.nxt_attn_last_error().decode())
    return n


def kv4_cache_empty(num_blocks: int, num_kv_heads: int, head_size: int, block_size: int, *,
                    device=None):
    """An uninitialised cache (of K, or of V): uint8 [num_blocks, num_kv_heads, page_bytes]."""
    import torch
    return torch.empty((num_blocks, num_kv_heads, kv4_page_bytes(head_size, block_size)),
                       dtype=torch.uint8, device=device)


def _on_current_device(*tensors) -> None:
    """Every tensor on the current GPU, whose stream and workspace a call uses."""
    import torch
    for t in tensors:
        if not t.is_cuda or t.device.index != torch.cuda.current_device():
            raise ValueError(f"tensor on {t.device}, not on the current GPU")


def _index_args(n: int, **tensors) -> None:
    """int32 contiguous arrays of n rows (None: not given)."""
    import torch
    for name, t in tensors.items():
        if t is None:
            continue
        if t.dtype != torch.int32 or not t.is_contiguous() or t.shape[0] != n:
            raise ValueError(f"{name} must be a contiguous int32 tensor of {n} rows")
        _on_current_device(t)


def _cache_args(key_cache, value_cache, kv_heads: int, head_size: int, block_size: int | None):
    """(block_size, block stride, head stride) of a cache pair; the page size
    gives the block size where the caller does not."""
    _on_current_device(key_cache, value_cache)
    if key_cache.shape[1] != kv_heads:
        raise ValueError(f"the cache has {key_cache.shape[1]} kv heads, not {kv_heads}")
    if key_cache.element_size() != 1 or value_cache.element_size() != 1:
        raise ValueError("a 4-bit cache is a uint8 tensor (kv4_cache_empty)")
    if key_cache.shape != value_cache.shape or key_cache.stride() != value_cache.stride():
        raise ValueError("key_cache and value_cache differ in shape or strides")
    page = key_cache.shape[2]
    if block_size is None:
        block_size = page // _page_bytes(head_size, 1)
    if page != _page_bytes(head_size, block_size) or key_cache.stride(2) != 1:
        raise ValueError(f"pages of {page} bytes do not hold whole tokens of head_size "
                         f"{head_size} and block_size {block_size}")
    return block_size, key_cache.stride(0), key_cache.stride(1)


def _rows_arg(name: str, key, value) -> None:
    if key.dtype != value.dtype or key.shape != value.shape:
        raise ValueError(f"{name}: key and value differ in dtype or shape")
    if not (key.is_contiguous() and value.is_contiguous()):
        raise ValueError(f"{name}: key and value rows must be contiguous")
    _on_current_device(key, value)


def paged_kv4_append(key_cache, value_cache, key, value, *, block_tables=None, positions=None,
                     slot_mapping=None, block_size: int | None = None, stream=None,
                     check: bool = True) -> int:
    """Quantise new K/V rows into the pages: with block_tables + positions
    (decode: row s is sequence s's token at positions[s]) through
    nxt_paged_kv4_append, or with slot_mapping (flat slot per row) through
    nxt_paged_kv4_write_slots.  No two rows of a call may have the same slot."""
    lib = _lib.backend()
    num_tokens, kvh, head_size = key.shape
    _rows_arg("paged_kv4_append", key, value)
    bs, bstride, hstride = _cache_args(key_cache, value_cache, kvh, head_size, block_size)
    _index_args(num_tokens, block_tables=block_tables, positions=positions,
                slot_mapping=slot_mapping)
    dtype, st = kv_dtype_of(key), _stream_handle(stream)
    if slot_mapping is not None:
        status = lib.nxt_paged_kv4_write_slots(
            _ptr(key_cache), _ptr(value_cache), _ptr(key), _ptr(value), _ptr(slot_mapping),
            num_tokens, kvh, head_size, bs, bstride, hstride, dtype, st)
    else:
        if block_tables is None or positions is None:
            raise ValueError("need block_tables and positions, or slot_mapping")
        status = lib.nxt_paged_kv4_append(
            _ptr(key_cache), _ptr(value_cache), _ptr(key), _ptr(value), _ptr(block_tables),
            _ptr(positions), num_tokens, kvh, head_size, block_tables.shape[1], bs, bstride,
            hstride, dtype, st)
    return _raise(lib, status, check)


def paged_kv4_read(key, value, key_cache, value_cache, slot_mapping, *,
                   block_size: int | None = None, stream=None, check: bool = True) -> int:
    """The values held in slot slot_mapping[i] into row i of key / value
    (nxt_paged_kv4_read_slots); a negative slot leaves its row as it was."""
    lib = _lib.backend()
    num_tokens, kvh, head_size = key.shape
    _rows_arg("paged_kv4_read", key, value)
    bs, bstride, hstride = _cache_args(key_cache, value_cache, kvh, head_size, block_size)
    _index_args(num_tokens, slot_mapping=slot_mapping)
    status = lib.nxt_paged_kv4_read_slots(
        _ptr(key), _ptr(value), _ptr(key_cache), _ptr(value_cache), _ptr(slot_mapping),
        num_tokens, kvh, head_size, bs, bstride, hstride, kv_dtype_of(key),
        _stream_handle(stream))
    return _raise(lib, status, check)


def paged_kv4_copy_slots(key_cache, value_cache, src_slots, dst_slots, *, head_size: int,
                         block_size: int | None = None, stream=None, check: bool = True) -> int:
    """Copy the rows of page slots src_slots[i] to dst_slots[i] (int32 device
    tensors) inside the caches (nxt_paged_kv4_copy_slots): the copy-on-write of
    a partly shared page at admission."""
    lib = _lib.backend()
    bs, bstride, hstride = _cache_args(key_cache, value_cache, key_cache.shape[1], head_size,
                                       block_size)
    _index_args(src_slots.shape[0], src_slots=src_slots, dst_slots=dst_slots)
    status = lib.nxt_paged_kv4_copy_slots(
        _ptr(key_cache), _ptr(value_cache), _ptr(src_slots), _ptr(dst_slots),
        src_slots.shape[0], key_cache.shape[1], head_size, bs, bstride, hstride,
        _stream_handle(stream))
    return _raise(lib, status, check)


def paged_attention_kv4(out, query, key_cache, value_cache, block_tables, seq_lens, *,
                        num_kv_heads: int, scale: float, block_size: int | None = None,
                        max_num_blocks_per_seq: int | None = None, stream=None,
                        check: bool = True) -> int:
    """Decode attention over a 4-bit cache (nxt_paged_attention_kv4): as
    paged_attention, with K and V the values that the cache holds."""
    lib = _lib.backend()
    num_seqs, num_heads, head_size = query.shape
    if out.dtype != query.dtype or out.shape != query.shape:
        raise ValueError("out and query differ in dtype or shape")
    if not (out.is_contiguous() and query.is_contiguous()):
        raise ValueError("query and out must be contiguous")
    bs, bstride, hstride = _cache_args(key_cache, value_cache, num_kv_heads, head_size,
                                       block_size)
    _on_current_device(query, out)
    _index_args(num_seqs, block_tables=block_tables, seq_lens=seq_lens)
    if max_num_blocks_per_seq is None:
        max_num_blocks_per_seq = block_tables.shape[1]
    status = lib.nxt_paged_attention_kv4(
        _ptr(out), _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(block_tables),
        _ptr(seq_lens), num_seqs, num_heads, head_size, num_kv_heads, ctypes.c_float(scale),
        max_num_blocks_per_seq, bs, bstride, hstride, kv_dtype_of(query), _stream_handle(stream))
    return _raise(lib, status, check)
