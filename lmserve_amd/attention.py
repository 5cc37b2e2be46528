"""Causal attention over the paged cache: what reads the pages that the writes fill.

Stands where the reference calls its prefill and decode wrappers behind the write
(runtime/worker/llm_worker/models/layers/attention.py:87-99): the same index tensors, the
same "NHD" cache `[num_pages, 2, page_size, H, D]`, one call for steps of single tokens,
of prefill chunks and of both. The leading pages that the requests of a batch share
(`shared_pages`) are read once for all of them.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .cache_ops import _on_device_of, _require_gpu, _stream_of
from .paged import _i32
from .quantized import _pages
from .rotary import _DTYPES

_raw_stream = torch._C._cuda_getCurrentRawStream


class PagedAttentionPlan:
    """Attention of a step's queries, its index arguments handed over ONCE.

    qo_indptr: int32 `[B + 1]`, the requests' rows in `query` (`cu_seqlens_q` of
      `build_write_index`); kv_indices, kv_indptr, kv_last_page_len: the block tables as
      the write takes them. All on the device.
    num_tokens: rows of `query` and `out` (a capacity; rows behind `qo_indptr[B]` are left
      as they were).
    shared_pages: the leading pages that the requests have in common, e.g.
      `index_prep.common_prefix_pages`. Requests that begin with other pages than the first are
      computed by themselves: the number changes the time and not the result.
    sm_scale: of the scores, `head_dim ** -0.5` when None.
    max_q_len: the most tokens a request has, if known: of help to the choice of kernels, not a limit.
    kv_dtype: `torch.float8_e4m3fn` for a cache in 8 bits (`lmserve_amd.quantized`), whose layers are
      `[num_pages, page_bytes]` of uint8; `dtype` is then the queries' and outputs'. `head_dim` and `page_size` are
      multiples of 16 with it.

    The step's work is laid out on the device at construction, by a small launch (two with shared pages) on the current
    stream; `build()` does it again after the index buffers were written for another step, and can
    be recorded with the runs into a hipGraph (keep the plan while that is replayed). Runs must be ordered after it. The
    plan keeps references to the index tensors; a step whose `qo_indptr` or `kv_indptr` decreases is not computed. Every run takes a workspace of its own from torch's allocator, so runs on
    different streams do not meet.
    """

    def __init__(self, qo_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
                 kv_last_page_len: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int,
                 dtype: torch.dtype, num_tokens: int, max_q_len: Optional[int] = None, shared_pages: int = 0,
                 sm_scale: Optional[float] = None, kv_layout: str = "NHD", kv_dtype: Optional[torch.dtype] = None):
        if kv_layout != "NHD":
            raise ValueError(f"kv_layout {kv_layout!r} is not supported (the reference uses 'NHD')")
        self._plan = None
        self.qo_indptr, self.kv_indices = _i32(qo_indptr, "qo_indptr"), _i32(kv_indices, "kv_indices")
        self.kv_indptr, self.kv_last_page_len = _i32(kv_indptr, "kv_indptr"), _i32(kv_last_page_len, "kv_last_page_len")
        # index tensors that are no dense arrays: the launches read copies, which `build` makes anew
        self._copies = [(copy, given) for copy, given in ((self.qo_indptr, qo_indptr), (self.kv_indices, kv_indices),
                                                          (self.kv_indptr, kv_indptr), (self.kv_last_page_len, kv_last_page_len))
                        if copy is not given]
        batch = self.kv_last_page_len.numel()
        if self.kv_indptr.numel() != batch + 1 or self.qo_indptr.numel() != batch + 1:
            raise ValueError("qo_indptr and kv_indptr must have batch_size + 1 entries")
        self.device = self.qo_indptr.device
        if any(t.device != self.device for t in (self.kv_indices, self.kv_indptr, self.kv_last_page_len)):
            raise ValueError("the index tensors must live on one device")
        kd = _DTYPES.get(dtype)
        if kd is None:
            raise TypeError(f"Unsupported dtype: {dtype}")
        if kv_dtype not in (None, dtype, torch.float8_e4m3fn):
            raise TypeError(f"Unsupported kv_dtype: {kv_dtype} (the cache holds {dtype} or float8_e4m3fn)")
        self.q8 = kv_dtype == torch.float8_e4m3fn
        self.dtype, self.num_tokens = dtype, int(num_tokens)
        self.Hq, self.H, self.D, self.page_size = int(num_heads), int(num_kv_heads), int(head_dim), int(page_size)
        lib = _lib.lib()
        handle = ctypes.c_void_p()
        create = lib.kvc_attention_plan_create_q8 if self.q8 else lib.kvc_attention_plan_create
        _lib.check(create(
            self.qo_indptr.data_ptr(), self.kv_indices.data_ptr(), self.kv_indptr.data_ptr(),
            self.kv_last_page_len.data_ptr(), batch, self.num_tokens, self.kv_indices.numel(), self.Hq, self.H,
            self.D, self.page_size, int(max_q_len or 0), int(shared_pages), self.D ** -0.5 if sm_scale is None else float(sm_scale), kd,
            ctypes.byref(handle)))
        self._plan = handle.value
        self._destroy = lib.kvc_attention_plan_destroy
        self._buffer = torch.empty(lib.kvc_attention_plan_bytes(self._plan), dtype=torch.uint8, device=self.device)
        self._workspace_bytes = lib.kvc_attention_workspace_bytes(self._plan)
        self._stream = _stream_of(self._buffer)      # whose allocator the buffer is from
        self._dev_index = self.device.index
        fast = _lib.fast()
        self._fast_run = (fast.attention_plan_run_q8 if self.q8 else fast.attention_plan_run) if fast else None
        self._dtype_code = fast.scalar_type_code(torch.empty(0, dtype=dtype)) if fast else -1
        self.build()

    def __del__(self):
        plan, self._plan = getattr(self, "_plan", None), None
        if plan:
            self._destroy(plan)

    def build(self) -> None:
        """Lay out the step that the index buffers hold (a small launch on the current stream, two with shared pages)."""
        with _on_device_of(self._buffer):
            self._used_here()
            for copy, given in self._copies:
                copy.copy_(given)
            _lib.check(_lib.lib().kvc_attention_plan_build(self._plan, self._buffer.data_ptr(), self._buffer.numel(),
                                                           _stream_of(self._buffer)))

    def _used_here(self) -> None:
        """What the plan owns stays allocated until the current stream's launches are done with it."""
        if _stream_of(self._buffer) != self._stream:
            stream = torch.cuda.current_stream()
            for owned in (self._buffer, *(copy for copy, _ in self._copies)):
                owned.record_stream(stream)

    def run(self, query: torch.Tensor, paged_kv_cache: torch.Tensor, out: Optional[torch.Tensor] = None,
            return_lse: bool = False, lse: Optional[torch.Tensor] = None):
        """One layer: `query [num_tokens, Hq, D]` (or `[num_tokens, Hq*D]`; rows may be slices
        of a fused projection) over `paged_kv_cache [num_pages, 2, page_size, H, D]`, or `[num_pages, page_bytes]` in 8 bits.
        Returns `out` in the query's shape, with `return_lse` also the fp32 `[num_tokens, Hq]` logarithms of the
        softmax sums. `out` / `lse` may be contiguous buffers of the caller's (`out` the query itself, but no other
        memory that is read); without one, rows
        behind the last request are not initialised. Launches on the current stream of the plan's device."""
        fast = self._fast_run
        if fast is not None and lse is None:
            # layouts checked and tensors allocated in C++; 1 = not a layout it knows: the checks below name what is wrong
            stream = _raw_stream(self._dev_index)
            if stream == self._stream:
                got = fast(self._plan, self.num_tokens, self.Hq, self.H, self.D, self.page_size, self._dtype_code,
                           self._dev_index, query, paged_kv_cache, out, return_lse, stream)
                if type(got) is not int:
                    return got
                if got < 0:
                    _lib.check(got)
        for t, n in ((query, "query"), (paged_kv_cache, "paged_kv_cache")):
            _require_gpu(t, n)
            if t.dtype != (torch.uint8 if self.q8 and t is paged_kv_cache else self.dtype) or t.device != self.device:
                raise TypeError(f"{n} must have the plan's dtype and device")
        T, row = self.num_tokens, self.Hq * self.D
        if query.dim() not in (2, 3) or query.shape[0] != T or query.numel() != T * row \
                or (query.dim() == 3 and query.shape[2] != self.D):
            raise ValueError(f"query must be [{T}, {self.Hq}, {self.D}] or [{T}, {row}]")
        q2 = query if query.dim() == 2 else query.flatten(1)
        if T and (q2.stride(1) != 1 or q2.data_ptr() % 16
                  or (T > 1 and (q2.stride(0) % 8 or q2.stride(0) < row))):
            q2 = q2.contiguous()
            if q2.data_ptr() % 16:
                q2 = q2.clone()
        shape, st = paged_kv_cache.shape, paged_kv_cache.stride()
        kv_row = self.H * self.D
        if self.q8:
            pages, page_size, page_stride = _pages(paged_kv_cache, self.H, self.D, "paged_kv_cache")
            if page_size != self.page_size:
                raise ValueError(f"paged_kv_cache has pages of {page_size} tokens, the plan of {self.page_size}")
        elif len(shape) != 5 or shape[1:] != (2, self.page_size, self.H, self.D):
            raise ValueError("paged_kv_cache must be [num_pages, 2, page_size, H, D]")
        else:
            pages = shape[0]
            page = 2 * self.page_size * kv_row
            page_stride = st[0] if pages > 1 else page
        if pages and not self.q8 and (st[4] != 1 or (st[3] != self.D and self.H > 1) or (st[2] != kv_row and self.page_size > 1)
                      or st[1] != page // 2):
            raise ValueError("every page of paged_kv_cache must be contiguous [2, page_size, H, D]")
        if out is None:
            out = torch.empty(query.shape, dtype=self.dtype, device=self.device)
        elif out.dtype != self.dtype or out.device != self.device or out.numel() != T * row or not out.is_contiguous():
            raise ValueError("out must be contiguous, of the query's size, dtype and device")
        if lse is None:
            lse = torch.empty((T, self.Hq), dtype=torch.float32, device=self.device) if return_lse else None
        elif lse.dtype != torch.float32 or lse.device != self.device or lse.numel() != T * self.Hq \
                or not lse.is_contiguous():
            raise ValueError("lse must be contiguous fp32 [num_tokens, num_heads] on the plan's device")
        if T:
            with _on_device_of(q2):
                stream = _stream_of(q2)
                self._used_here()
                workspace = torch.empty(self._workspace_bytes, dtype=torch.uint8, device=self.device)
                run = _lib.lib().kvc_attention_plan_run_q8 if self.q8 else _lib.lib().kvc_attention_plan_run
                _lib.check(run(
                    self._plan, q2.data_ptr(), q2.stride(0) if T > 1 else row, paged_kv_cache.data_ptr(),
                    page_stride, pages, out.data_ptr(), None if lse is None else lse.data_ptr(),
                    workspace.data_ptr(), workspace.numel(), stream))
        return (out, lse) if return_lse else out


def paged_attention(query: torch.Tensor, paged_kv_cache: torch.Tensor, qo_indptr: torch.Tensor,
                    kv_indices: torch.Tensor, kv_indptr: torch.Tensor, kv_last_page_len: torch.Tensor,
                    max_q_len: Optional[int] = None, shared_pages: int = 0, sm_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False, kv_layout: str = "NHD",
                    num_kv_heads: Optional[int] = None):
    """`PagedAttentionPlan` made and run once: attention of one layer with index tensors that
    serve no other (a model's layers share a plan). Arguments and results are the plan's. A cache
    `[num_pages, page_bytes]` of uint8 is one in 8 bits: `query` is then `[T, Hq, D]`, and `num_kv_heads` has to be given."""
    if isinstance(paged_kv_cache, torch.Tensor) and paged_kv_cache.dtype == torch.uint8:
        return _paged_attention_q8(query, paged_kv_cache, qo_indptr, kv_indices, kv_indptr, kv_last_page_len, max_q_len,
                                   shared_pages, sm_scale, out, return_lse, kv_layout, num_kv_heads)
    fast = _lib.fast_entry("paged_attention")
    if fast is not None and kv_layout == "NHD" and isinstance(paged_kv_cache, torch.Tensor) and paged_kv_cache.is_cuda \
            and num_kv_heads is None:
        # common layouts: checked and launched from C++ (1 = not one of them: fall through)
        dev = paged_kv_cache.device.index
        got = fast(query, paged_kv_cache, qo_indptr, kv_indices, kv_indptr, kv_last_page_len, max_q_len or 0, shared_pages,
                   (paged_kv_cache.shape[-1] or 1) ** -0.5 if sm_scale is None else sm_scale, out, return_lse, dev,
                   _raw_stream(dev))
        if type(got) is not int:
            return got
        if got < 0:
            _lib.check(got)
    for t, n in ((query, "query"), (paged_kv_cache, "paged_kv_cache")):
        _require_gpu(t, n)
    if paged_kv_cache.dim() != 5 or paged_kv_cache.shape[1] != 2:
        raise ValueError("paged_kv_cache must be [num_pages, 2, page_size, H, D]")
    _, _, page_size, H, D = paged_kv_cache.shape
    if num_kv_heads not in (None, H):
        raise ValueError(f"num_kv_heads is {num_kv_heads}, the cache has {H}")
    if query.dim() not in (2, 3) or D == 0 or query.shape[-1] % D:
        raise ValueError("query must be [T, Hq, D] or [T, Hq*D]")
    heads = query.shape[1] if query.dim() == 3 else query.shape[1] // D
    plan = PagedAttentionPlan(qo_indptr, kv_indices, kv_indptr, kv_last_page_len, heads, H, D, page_size, query.dtype,
                              query.shape[0], max_q_len=max_q_len, shared_pages=shared_pages, sm_scale=sm_scale,
                              kv_layout=kv_layout)
    return plan.run(query, paged_kv_cache, out=out, return_lse=return_lse)


def _paged_attention_q8(query, paged_kv_cache, qo_indptr, kv_indices, kv_indptr, kv_last_page_len, max_q_len, shared_pages,
                        sm_scale, out, return_lse, kv_layout, num_kv_heads):
    fast = _lib.fast_entry("paged_attention")
    if fast is not None and num_kv_heads is not None and kv_layout == "NHD" and paged_kv_cache.is_cuda and query.dim() == 3:
        # as for 16 bits
        dev = paged_kv_cache.device.index
        got = fast(query, paged_kv_cache, qo_indptr, kv_indices, kv_indptr, kv_last_page_len, max_q_len or 0, shared_pages,
                   (query.shape[2] or 1) ** -0.5 if sm_scale is None else sm_scale, out, return_lse, dev, _raw_stream(dev),
                   num_kv_heads)
        if type(got) is not int:
            return got
        if got < 0:
            _lib.check(got)
    for t, n in ((query, "query"), (paged_kv_cache, "paged_kv_cache")):
        _require_gpu(t, n)
    if query.dim() != 3 or num_kv_heads is None:
        raise ValueError("over a cache in 8 bits query must be [T, Hq, D] and num_kv_heads given")
    _, heads, D = query.shape
    _, page_size, _ = _pages(paged_kv_cache, int(num_kv_heads), D, "paged_kv_cache")
    plan = PagedAttentionPlan(qo_indptr, kv_indices, kv_indptr, kv_last_page_len, heads, num_kv_heads, D, page_size, query.dtype,
                              query.shape[0], max_q_len=max_q_len, shared_pages=shared_pages, sm_scale=sm_scale,
                              kv_layout=kv_layout, kv_dtype=torch.float8_e4m3fn)
    return plan.run(query, paged_kv_cache, out=out, return_lse=return_lse)
