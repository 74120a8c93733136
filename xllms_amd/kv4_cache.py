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

from . import _lib
from .paged_attention import NXT_ATTN_OK, PagedAttentionError, _stream_handle, kv_dtype_of

GROUP = 32  # channels that share a range
TILE = 16   # tokens of a tile: the smallest block_size
_MAX_STRIDE = 2**31 - 1  # the C calls take strides as int, in bytes

_int32 = _uint8 = _device_of = None  # of torch, which is imported on first use


def _current_device() -> int:
    """Index of the current GPU (-2 before torch has initialised one, which no
    tensor's get_device() is).  The checks here are what a small call's time
    goes into: plain attribute reads, no Device objects."""
    global _int32, _uint8, _device_of
    if _device_of is None:
        import torch
        if not torch.cuda.is_initialized():
            return -2
        _int32, _uint8, _device_of = torch.int32, torch.uint8, torch.cuda.current_device
    return _device_of()


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


def _pair(name: str, device: int, a, b) -> None:
    """Two row tensors: the same dtype and shape, contiguous, on the current GPU
    (whose stream and workspace a call uses)."""
    if a.get_device() != device or b.get_device() != device:
        raise ValueError(f"{name}: tensors on {a.device} and {b.device}, not on the current GPU")
    if a.dtype != b.dtype or a.shape != b.shape:
        raise ValueError(f"{name}: the row tensors differ in dtype or shape")
    if not (a.is_contiguous() and b.is_contiguous()):
        raise ValueError(f"{name}: rows must be contiguous")


def _index(name: str, device: int, t, n: int, dims: int = 1) -> int:
    """Address of an int32 array of n entries (of dims 2, rows)."""
    if t.dtype is not _int32 or t.dim() != dims or t.shape[0] != n or \
            not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {dims} dimension(s), the "
                         f"first of {n}, on the current GPU")
    return t.data_ptr()


def _cache_args(device: int, key_cache, value_cache, kv_heads: int, head_size: int,
                block_size: int | None):
    """(block_size, block stride, head stride) of a cache pair; the page size
    gives the block size where the caller does not."""
    if key_cache.get_device() != device or value_cache.get_device() != device:
        raise ValueError(f"caches on {key_cache.device} and {value_cache.device}, not on the "
                         "current GPU")
    shape, stride = key_cache.shape, key_cache.stride()
    if key_cache.dtype is not _uint8 or value_cache.dtype is not _uint8 or len(shape) != 3:
        raise ValueError("a 4-bit cache is a uint8 tensor of 3 dimensions (kv4_cache_empty)")
    if shape != value_cache.shape or stride != value_cache.stride():
        raise ValueError("key_cache and value_cache differ in shape or strides")
    if stride[0] > _MAX_STRIDE or stride[1] > _MAX_STRIDE:
        raise ValueError(f"strides of {stride[0]} and {stride[1]} bytes: at most {_MAX_STRIDE}")
    if shape[1] != kv_heads:
        raise ValueError(f"the cache has {shape[1]} kv heads, not {kv_heads}")
    page = shape[2]
    if head_size <= 0:
        raise ValueError(f"head_size {head_size}")
    if block_size is None:
        block_size = page // _page_bytes(head_size, 1)
    if page != _page_bytes(head_size, block_size) or stride[2] != 1:
        raise ValueError(f"pages of {page} bytes do not hold whole tokens of head_size "
                         f"{head_size} and block_size {block_size}")
    return block_size, stride[0], stride[1]


def paged_kv4_append(key_cache, value_cache, key, value, *, block_tables=None, positions=None,
                     slot_mapping=None, block_size: int | None = None, stream=None,
                     check: bool = True) -> int:
    """Quantise new K/V rows into the pages: with block_tables + positions
    (decode: row s is sequence s's token at positions[s]) through
    nxt_paged_kv4_append, or with slot_mapping (flat slot per row) through
    nxt_paged_kv4_write_slots.  No two rows of a call may have the same slot."""
    lib, dev = _lib.backend(), _current_device()
    num_tokens, kvh, head_size = key.shape
    _pair("paged_kv4_append", dev, key, value)
    bs, bstride, hstride = _cache_args(dev, key_cache, value_cache, kvh, head_size, block_size)
    dtype, st = kv_dtype_of(key), _stream_handle(stream)
    if slot_mapping is not None:
        status = lib.nxt_paged_kv4_write_slots(
            key_cache.data_ptr(), value_cache.data_ptr(), key.data_ptr(), value.data_ptr(),
            _index("slot_mapping", dev, slot_mapping, num_tokens), num_tokens, kvh, head_size, bs,
            bstride, hstride, dtype, st)
    else:
        if block_tables is None or positions is None:
            raise ValueError("need block_tables and positions, or slot_mapping")
        status = lib.nxt_paged_kv4_append(
            key_cache.data_ptr(), value_cache.data_ptr(), key.data_ptr(), value.data_ptr(),
            _index("block_tables", dev, block_tables, num_tokens, 2),
            _index("positions", dev, positions, num_tokens), num_tokens, kvh, head_size,
            block_tables.shape[1], bs, bstride, hstride, dtype, st)
    return _raise(lib, status, check)


def paged_kv4_read(key, value, key_cache, value_cache, slot_mapping, *,
                   block_size: int | None = None, stream=None, check: bool = True) -> int:
    """The values held in slot slot_mapping[i] into row i of key / value
    (nxt_paged_kv4_read_slots); a negative slot leaves its row as it was."""
    lib, dev = _lib.backend(), _current_device()
    num_tokens, kvh, head_size = key.shape
    _pair("paged_kv4_read", dev, key, value)
    bs, bstride, hstride = _cache_args(dev, key_cache, value_cache, kvh, head_size, block_size)
    status = lib.nxt_paged_kv4_read_slots(
        key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
        _index("slot_mapping", dev, slot_mapping, num_tokens), num_tokens, kvh, head_size, bs,
        bstride, hstride, kv_dtype_of(key), _stream_handle(stream))
    return _raise(lib, status, check)


def paged_kv4_copy_slots(key_cache, value_cache, src_slots, dst_slots, *, head_size: int,
                         block_size: int | None = None, stream=None, check: bool = True) -> int:
    """Copy the rows of page slots src_slots[i] to dst_slots[i] (int32 device
    tensors) inside the caches (nxt_paged_kv4_copy_slots): the copy-on-write of
    a partly shared page at admission."""
    lib, dev = _lib.backend(), _current_device()
    kvh, n = key_cache.shape[1], src_slots.shape[0]
    bs, bstride, hstride = _cache_args(dev, key_cache, value_cache, kvh, head_size, block_size)
    status = lib.nxt_paged_kv4_copy_slots(
        key_cache.data_ptr(), value_cache.data_ptr(), _index("src_slots", dev, src_slots, n),
        _index("dst_slots", dev, dst_slots, n), n, kvh, head_size, bs, bstride, hstride,
        _stream_handle(stream))
    return _raise(lib, status, check)


def paged_attention_kv4(out, query, key_cache, value_cache, block_tables, seq_lens, *,
                        num_kv_heads: int, scale: float, block_size: int | None = None,
                        stream=None, check: bool = True) -> int:
    """Decode attention over a 4-bit cache (nxt_paged_attention_kv4): as
    paged_attention, with K and V the values that the cache holds."""
    lib, dev = _lib.backend(), _current_device()
    num_seqs, num_heads, head_size = query.shape
    _pair("paged_attention_kv4", dev, out, query)
    bs, bstride, hstride = _cache_args(dev, key_cache, value_cache, num_kv_heads, head_size,
                                       block_size)
    tables = _index("block_tables", dev, block_tables, num_seqs, 2)
    status = lib.nxt_paged_attention_kv4(
        out.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
        tables, _index("seq_lens", dev, seq_lens, num_seqs), num_seqs, num_heads, head_size,
        num_kv_heads, float(scale), block_tables.shape[1], bs, bstride, hstride,
        kv_dtype_of(query), _stream_handle(stream))
    return _raise(lib, status, check)
