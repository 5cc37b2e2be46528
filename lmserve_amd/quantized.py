"""The paged cache in 8 bits: quantised as it is written, read back, its layout.

Beside the 16-bit write of the reference's call site
(runtime/worker/llm_worker/models/layers/attention.py:76-85): the same slots and index
tensors, a cache of half the bytes. A pool is `[L, num_blocks, block_bytes]` of uint8, a
block `block_size / 16` groups of 16 tokens, each with its codes (e4m3) and one exponent for
every head and for K and V (include/kvcache.h has the layout). Blocks move as bytes:
`copy_blocks`, `gather_blocks`, `KVWorker` and the disk tier take such a pool as it is.

A group's exponent is that of the largest value written into it. A request's tokens come in the order
of their positions: a call that begins at a group's first place begins the group anew, and one that goes on with it
rounds what is there to a greater exponent where it has to. It stores the group's other tokens again, so whatever reads
or moves a block that is still being filled is ordered with the writes into it.

`PagedAttentionPlan(kv_dtype=torch.float8_e4m3fn)` and `paged_attention` attend to such a cache.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .cache_ops import _on_device_of, _require_gpu, _slot_args, _stream_of
from .kv_pool import CachePlan
from .paged import _paged_common
from .rotary import _DTYPES

GROUP = 16      # tokens that share an exponent
_raw_stream = torch._C._cuda_getCurrentRawStream
_fast_entry = _lib.fast_entry
_READ_DTYPES = {torch.bfloat16: _lib.KVC_DTYPE_BF16, torch.float16: _lib.KVC_DTYPE_F16}


def q8_page_bytes(num_kv_heads: int, head_dim: int, page_size: int) -> int:
    """Bytes of a page (block) of one layer. `head_dim` is a multiple of 16 up to 256, `page_size` a multiple of 16."""
    got = _lib.lib().kvc_q8_page_bytes(int(num_kv_heads), int(head_dim), int(page_size))
    if got < 0:
        _lib.check(got)
    return got


def plan_q8_cache(gpu_cache_size: int, host_cache_size: int, disk_cache_size: int, num_layers: int,
                  num_kv_heads: int, head_dim: int, block_size: int) -> CachePlan:
    """`plan_cache` for 8-bit blocks: how many each tier's bytes hold. `kv_block_size` is half
    a block of one layer, its exponents and padding included."""
    block = q8_page_bytes(num_kv_heads, head_dim, block_size)
    per_block = num_layers * block
    return CachePlan(block // 2, int(gpu_cache_size) // per_block, int(host_cache_size) // per_block,
                     int(disk_cache_size) // per_block)


def allocate_q8_kv_caches(num_layers: int, num_gpu_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                          device="cuda") -> torch.Tensor:
    """The pool `[L, num_gpu_blocks, block_bytes]` of uint8, uninitialised as `allocate_kv_caches` leaves its own."""
    return torch.empty(num_layers, num_gpu_blocks, q8_page_bytes(num_kv_heads, head_dim, block_size),
                       dtype=torch.uint8, device=device)


def _pages(cache: torch.Tensor, num_kv_heads: int, head_dim: int, name: str) -> Tuple[int, int, int]:
    """(pages, page_size, bytes from page to page) of one layer's cache `[num_pages, page_bytes]`."""
    _require_gpu(cache, name)
    if cache.dtype != torch.uint8:
        raise TypeError(f"{name} must be uint8 (an 8-bit cache)")
    if cache.dim() != 2 or (cache.shape[1] > 1 and cache.stride(1) != 1):
        raise ValueError(f"{name} must be [num_pages, page_bytes] with contiguous pages")
    group = q8_page_bytes(num_kv_heads, head_dim, GROUP)
    if cache.shape[1] == 0 or cache.shape[1] % group:
        raise ValueError(f"{name} has pages of {cache.shape[1]} bytes: {num_kv_heads} heads of {head_dim} take a multiple of {group}")
    return cache.shape[0], cache.shape[1] // group * GROUP, cache.stride(0) if cache.shape[0] > 1 else cache.shape[1]


def _token_rows(t: torch.Tensor, name: str, num_kv_heads: int, head_dim: int) -> Tuple[torch.Tensor, int]:
    """Rows `[T, H, D]` or `[T, H*D]`, dense inside a token and aligned to 16 bytes (or a copy that is), and their stride."""
    _require_gpu(t, name)
    row = num_kv_heads * head_dim
    if t.dim() == 3 and t.shape[1:] == (num_kv_heads, head_dim):
        dense = t.stride(2) == 1 and (num_kv_heads == 1 or t.stride(1) == head_dim)
    elif t.dim() == 2 and t.shape[1] == row:
        dense = t.stride(1) == 1
    else:
        raise ValueError(f"{name} must be [num_tokens, {num_kv_heads}, {head_dim}] or [num_tokens, {row}]")
    many = t.shape[0] > 1
    if not dense or t.data_ptr() % 16 or (many and (t.stride(0) % 8 or t.stride(0) < row)):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t, t.stride(0) if t.shape[0] > 1 else row


def _heads_of(key: torch.Tensor, name: str) -> Tuple[int, int]:
    if key.dim() != 3:
        raise ValueError(f"{name} must be [num_tokens, num_kv_heads, head_dim]")
    return key.shape[1], key.shape[2]


def _dtype_code(*tensors: torch.Tensor) -> int:
    dtype = tensors[0].dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"Unsupported dtype: {dtype} (keys and values are bf16 or f16)")
    if any(t.dtype != dtype for t in tensors):
        raise TypeError("key and value must share one dtype")
    return _DTYPES[dtype]


def _same_device(cache: torch.Tensor, *tensors: torch.Tensor) -> None:
    if any(t.device != cache.device for t in tensors):
        raise ValueError("all tensors must live on the cache's device")


def reshape_and_cache_q8(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
                         slot_mapping: torch.Tensor) -> None:
    """`reshape_and_cache` into one layer of an 8-bit pool: token `i` goes to place `slot % block_size` of
    block `slot // block_size`, `slot = slot_mapping[i]`; a slot outside the cache is skipped.

    key, value: `[T, H, D]`, bf16 or f16 (rows may be slices of a fused projection); kv_cache: uint8
    `[num_blocks, block_bytes]`, `kv_caches[l]` of the pool; slot_mapping: `[T]` int32/int64 on the device.
    """
    fast = _fast_entry("write_q8")
    if fast is not None and isinstance(kv_cache, torch.Tensor) and kv_cache.is_cuda:
        # common layouts: checked and launched from C++ (1 = not one of them: fall through)
        dev = kv_cache.device.index
        rc = fast(key, value, kv_cache, dev, _raw_stream(dev), slot_mapping)
        if rc == 0:
            return
        if rc < 0:
            _lib.check(rc)
    H, D = _heads_of(key, "key")
    pages, page_size, stride = _pages(kv_cache, H, D, "kv_cache")
    _require_gpu(slot_mapping, "slot_mapping")
    key, k_stride = _token_rows(key, "key", H, D)
    value, v_stride = _token_rows(value, "value", H, D)
    code = _dtype_code(key, value)
    slot_mapping, slot_bytes = _slot_args(slot_mapping)
    _same_device(kv_cache, key, value, slot_mapping)
    tokens = slot_mapping.numel()
    if tokens != key.shape[0] or tokens != value.shape[0]:
        raise ValueError("key, value and slot_mapping must have one row for every token")
    if tokens == 0 or pages == 0:
        return
    with _on_device_of(kv_cache):
        _lib.check(_lib.lib().kvc_reshape_and_cache_q8(
            key.data_ptr(), value.data_ptr(), kv_cache.data_ptr(), slot_mapping.data_ptr(), slot_bytes, tokens, H, D,
            page_size, k_stride, v_stride, stride, pages, code, _stream_of(kv_cache)))


def append_paged_kv_cache_q8(append_key: torch.Tensor, append_value: torch.Tensor, batch_indices: torch.Tensor,
                             positions: torch.Tensor, paged_kv_cache: torch.Tensor, kv_indices: torch.Tensor,
                             kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor, kv_layout: str = "NHD") -> None:
    """`append_paged_kv_cache` into one layer of an 8-bit pool, `[num_pages, page_bytes]` of uint8: token `i` to
    place `p % page_size` of page `kv_indices[kv_indptr[b] + p // page_size]`, `b = batch_indices[i]`, `p = positions[i]`."""
    fast = _fast_entry("write_q8")
    if fast is not None and kv_layout == "NHD" and isinstance(paged_kv_cache, torch.Tensor) and paged_kv_cache.is_cuda \
            and kv_last_page_len.is_cuda and kv_last_page_len.dtype == torch.int32:
        # common layouts: checked and launched from C++ (1 = not one of them: fall through)
        dev = paged_kv_cache.device.index
        rc = fast(append_key, append_value, paged_kv_cache, dev, _raw_stream(dev), batch_indices, positions, kv_indices, kv_indptr)
        if rc == 0:
            return
        if rc < 0:
            _lib.check(rc)
    H, D = _heads_of(append_key, "append_key")
    pages, page_size, stride = _pages(paged_kv_cache, H, D, "paged_kv_cache")
    batch_indices, positions, kv_indices, kv_indptr, kv_last_page_len = _paged_common(
        append_key, append_value, batch_indices, positions, kv_indices, kv_indptr, kv_last_page_len, kv_layout)
    key, k_stride = _token_rows(append_key, "append_key", H, D)
    value, v_stride = _token_rows(append_value, "append_value", H, D)
    code = _dtype_code(key, value)
    _same_device(paged_kv_cache, key, value, batch_indices, positions, kv_indices, kv_indptr)
    nnz = batch_indices.numel()
    if key.shape[0] < nnz or value.shape[0] < nnz:
        raise ValueError("fewer key/value rows than index entries")
    if nnz == 0 or pages == 0:
        return
    with _on_device_of(paged_kv_cache):
        _lib.check(_lib.lib().kvc_append_paged_kv_cache_q8(
            key.data_ptr(), value.data_ptr(), batch_indices.data_ptr(), positions.data_ptr(), paged_kv_cache.data_ptr(),
            kv_indices.data_ptr(), kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), nnz, kv_indptr.numel() - 1,
            kv_indices.numel(), H, D, page_size, k_stride, v_stride, stride, pages, code, _stream_of(paged_kv_cache)))


def _outputs(cache: torch.Tensor, tokens: int, H: int, D: int, dtype: torch.dtype, key: Optional[torch.Tensor],
             value: Optional[torch.Tensor]):
    out = []
    for t, name in ((key, "key"), (value, "value")):
        if t is None:
            t = torch.empty(tokens, H, D, dtype=dtype, device=cache.device)
        rows, stride = _token_rows(t, name, H, D)
        if rows is not t or t.dtype != dtype or t.shape[0] < tokens:
            raise ValueError(f"{name} must hold {tokens} rows of {dtype}, dense and aligned to 16 bytes")
        out += [t, stride]
    _same_device(cache, out[0], out[2])
    return out


def read_cache_q8(kv_cache: torch.Tensor, slot_mapping: torch.Tensor, num_kv_heads: int, head_dim: int,
                  dtype: torch.dtype = torch.bfloat16, key: Optional[torch.Tensor] = None,
                  value: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values at the slots of one layer's 8-bit cache as `[T, H, D]` rows of `dtype` (bf16 or f16):
    the way back of `reshape_and_cache_q8`, slots in any order. `key` / `value` may be buffers of the
    caller's; rows of slots outside the cache are left as they were."""
    H, D = int(num_kv_heads), int(head_dim)
    fast = _fast_entry("read_q8")
    if fast is not None and key is None and value is None and dtype in _READ_DTYPES and kv_cache.is_cuda:
        # common layouts: checked and launched from C++ (1 = not one of them: fall through)
        dev = kv_cache.device.index
        got = fast(kv_cache, H, D, _READ_DTYPES[dtype], dev, _raw_stream(dev), slot_mapping)
        if type(got) is not int:
            return got
        if got < 0:
            _lib.check(got)
    pages, page_size, stride = _pages(kv_cache, H, D, "kv_cache")
    _require_gpu(slot_mapping, "slot_mapping")
    slot_mapping, slot_bytes = _slot_args(slot_mapping)
    tokens = slot_mapping.numel()
    key, k_stride, value, v_stride = _outputs(kv_cache, tokens, H, D, dtype, key, value)
    code = _dtype_code(key, value)
    _same_device(kv_cache, slot_mapping)
    if tokens and pages:
        with _on_device_of(kv_cache):
            _lib.check(_lib.lib().kvc_read_cache_q8(
                kv_cache.data_ptr(), slot_mapping.data_ptr(), slot_bytes, key.data_ptr(), value.data_ptr(), tokens, H, D,
                page_size, k_stride, v_stride, stride, pages, code, _stream_of(kv_cache)))
    return key, value


def read_paged_kv_cache_q8(batch_indices: torch.Tensor, positions: torch.Tensor, paged_kv_cache: torch.Tensor,
                           kv_indices: torch.Tensor, kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor,
                           num_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                           key: Optional[torch.Tensor] = None, value: Optional[torch.Tensor] = None,
                           kv_layout: str = "NHD") -> Tuple[torch.Tensor, torch.Tensor]:
    """`read_cache_q8` by the page table: the way back of `append_paged_kv_cache_q8`, tokens in any order."""
    H, D = int(num_kv_heads), int(head_dim)
    fast = _fast_entry("read_q8")
    if fast is not None and kv_layout == "NHD" and key is None and value is None and dtype in _READ_DTYPES and paged_kv_cache.is_cuda \
            and kv_last_page_len.is_cuda and kv_last_page_len.dtype == torch.int32:
        # common layouts: checked and launched from C++ (1 = not one of them: fall through)
        dev = paged_kv_cache.device.index
        got = fast(paged_kv_cache, H, D, _READ_DTYPES[dtype], dev, _raw_stream(dev), batch_indices, positions, kv_indices, kv_indptr)
        if type(got) is not int:
            return got
        if got < 0:
            _lib.check(got)
    pages, page_size, stride = _pages(paged_kv_cache, H, D, "paged_kv_cache")
    batch_indices, positions, kv_indices, kv_indptr, kv_last_page_len = _paged_common(
        None, None, batch_indices, positions, kv_indices, kv_indptr, kv_last_page_len, kv_layout)
    nnz = batch_indices.numel()
    key, k_stride, value, v_stride = _outputs(paged_kv_cache, nnz, H, D, dtype, key, value)
    code = _dtype_code(key, value)
    _same_device(paged_kv_cache, batch_indices, positions, kv_indices, kv_indptr)
    if nnz and pages:
        with _on_device_of(paged_kv_cache):
            _lib.check(_lib.lib().kvc_read_paged_kv_cache_q8(
                batch_indices.data_ptr(), positions.data_ptr(), paged_kv_cache.data_ptr(), kv_indices.data_ptr(),
                kv_indptr.data_ptr(), kv_last_page_len.data_ptr(), key.data_ptr(), value.data_ptr(), nnz,
                kv_indptr.numel() - 1, kv_indices.numel(), H, D, page_size, k_stride, v_stride, stride, pages, code,
                _stream_of(paged_kv_cache)))
    return key, value
