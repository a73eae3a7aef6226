"""Bounded paged KV cache (the q3_cache_* C ABI, csrc/cache*.cu): the buffers of
one layer's cache for several sequences, on which :class:`B200Backend`'s
``cache_append``, ``cache_attention`` and ``cache_evict`` work."""
from __future__ import annotations

import ctypes as C

from ._lib import CacheDesc, check, lib


class PagedCache:
    """One layer's cache of ``rows`` sequences over caller-owned CUDA tensors:

    k_pages, v_pages  bf16 [num_pages, kv_heads, 64, 128]
    page_tables       int32 [rows, >= ceil(max_len / 64)]: slot s of sequence r is
                      row s % 64 of page page_tables[r, s // 64]
    weights           fp32 [rows, kv_heads, >= max_len]: attention received by a slot
    positions         int32, as weights: the token position a slot holds

    weights and positions may both be None (no accumulation, no eviction).
    max_len, the slots a sequence may hold, defaults to what the page tables and
    weights cover.  The handle keeps the tensors alive.  Calls on one cache are
    ordered by the caller: one stream, or events.  A graph that captured calls
    on a cache writes the cache's own state words when it is replayed: keep the
    PagedCache until the graph is dropped.  (Without a graph it may be dropped
    while its last calls run, on any stream; the tensors given to it follow
    torch's rules for tensors used on several streams.)"""

    def __init__(self, k_pages, v_pages, page_tables, weights=None, positions=None, max_len: int | None = None):
        import torch

        dev = k_pages.device
        if dev.type != "cuda":
            raise ValueError("PagedCache: CUDA tensors required")
        if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
            raise ValueError("PagedCache: k_pages and v_pages must be [num_pages, kv_heads, 64, 128]")
        if (k_pages.dtype != torch.bfloat16 or v_pages.dtype != torch.bfloat16 or not k_pages.is_contiguous()
                or not v_pages.is_contiguous()):
            raise ValueError("PagedCache: k_pages and v_pages must be contiguous bf16 tensors")
        if page_tables.dtype != torch.int32 or page_tables.dim() != 2 or page_tables.stride(1) != 1:
            raise ValueError("PagedCache: page_tables must be int32 [rows, pages] with contiguous rows")
        rows, kvh = page_tables.shape[0], k_pages.shape[1]
        cover = page_tables.shape[1] * k_pages.shape[2]
        if (weights is None) != (positions is None):
            raise ValueError("PagedCache: weights and positions go together")
        if weights is not None:
            for t, want in ((weights, torch.float32), (positions, torch.int32)):
                if t.dtype != want or t.dim() != 3 or tuple(t.shape[:2]) != (rows, kvh):
                    raise ValueError("PagedCache: weights (fp32) and positions (int32) must be [rows, kv_heads, slots]")
                self._check_slots(t, weights)
            cover = min(cover, weights.shape[2])
        for t in (v_pages, page_tables, weights, positions):
            if t is not None and t.device != dev:
                raise ValueError("PagedCache: all tensors must be on one device")
        max_len = cover if max_len is None else max_len
        if not 1 <= max_len <= cover:
            raise ValueError(f"PagedCache: max_len must be 1 .. {cover}, what the page tables and weights cover")
        self.k_pages, self.v_pages, self.page_tables = k_pages, v_pages, page_tables
        self.weights, self.positions = weights, positions
        self.device, self.rows, self.kv_heads, self.max_len = dev, rows, kvh, max_len
        self.state = torch.zeros(4, dtype=torch.int32, device=dev)
        d = CacheDesc(k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0], page_tables.data_ptr(),
                      page_tables.stride(0) if rows > 1 else page_tables.shape[1],
                      weights.data_ptr() if weights is not None else None,
                      positions.data_ptr() if positions is not None else None,
                      weights.stride(1) if weights is not None else 0, rows, max_len, kvh, k_pages.shape[3],
                      k_pages.shape[2], self.state.data_ptr())
        h = C.c_void_p()
        check(lib().q3_cache_create(C.byref(d), dev.index, C.byref(h)))
        self.h = h
        self._empty, self._uint8, self._need = torch.empty, torch.uint8, {}
        # the zeroed state is there before any stream's kernels can reach it
        stream = torch.cuda.current_stream(dev)
        stream.synchronize()
        self._streams = {stream.cuda_stream}  # that the allocator knows to use the state

    @staticmethod
    def _check_slots(t, like):
        if t.stride(2) != 1 or t.stride(0) != t.shape[1] * t.stride(1) or t.stride() != like.stride():
            raise ValueError("PagedCache: weights and positions must have contiguous slots and evenly spaced heads, "
                             "laid out alike")

    def _used_on(self, stream):
        """The first call on `stream`, the current one, which is not that of the construction: kernels there write the
        state words, so the allocator keeps their memory until that stream has passed what it held when this cache was
        dropped.  A captured call runs when its graph is replayed, on any stream: the cache outlives the graph."""
        import torch

        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                return
        self.state.record_stream(torch.cuda.current_stream(self.device))
        self._streams.add(stream)

    def _scratch(self, call):
        """A workspace for one call, ("attention", q_heads, accumulate) or ("evict", keep), from torch's
        stream-ordered allocator: calls on different streams and captured graphs never share one."""
        need = self._need.get(call)
        if need is None:
            if call[0] == "attention":
                need = lib().q3_cache_attention_workspace_bytes(self.h, call[1], call[2])
            else:
                need = lib().q3_cache_evict_workspace_bytes(self.h, call[1])
            if len(self._need) < 1024:
                self._need[call] = need
        return self._empty(max(need, 16), dtype=self._uint8, device=self.device)

    def sync(self):
        """Waits for the current stream and raises if a kernel met a value out of range in device memory."""
        import torch

        check(lib().q3_cache_sync(self.h, torch.cuda.current_stream(self.device).cuda_stream))

    def close(self):
        if getattr(self, "h", None):
            lib().q3_cache_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
