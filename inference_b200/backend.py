"""B200Backend: the reference's Backend operator interface
(src/lib/backend/backend.hpp:16-42) over the op-level C ABI.

Tensors are torch CUDA tensors (torch supplies device memory and the
stream: plumbing only); every op runs a kernel of libq3_sm100a.so.  Method
names, argument order, in-place and aliasing behaviour follow backend.hpp, so
tests read like the reference's testing/tests/*.cpp.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import check, lib


def _torch():
    import torch

    return torch


def _p(t) -> int:
    return t.data_ptr()


class RopeCache:
    """backend::RopeCache (rope_cache.hpp:14-21): fp32 cos/sin [max_pos, hd/2]."""

    def __init__(self, cosine, sine):
        self.cosine, self.sine = cosine, sine


class B200Backend:
    def __init__(self, device: int = 0):
        torch = _torch()
        self.device = torch.device("cuda", device)
        self._ws = None
        self._idx = None
        self._bf16, self._f32, self._i32 = torch.bfloat16, torch.float32, torch.int32
        # the current stream of a device as a cudaStream_t, without the Python object around it
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)

    def _stream(self) -> int:
        return _torch().cuda.current_stream(self.device).cuda_stream

    def make_rope_cache(self, max_position: int, head_size: int, theta: float) -> RopeCache:
        torch = _torch()
        c = np.empty((max_position, head_size // 2), np.float32)
        s = np.empty_like(c)
        check(lib().q3_rope_tables(max_position, head_size, theta, c.ctypes.data, s.ctypes.data))
        return RopeCache(torch.from_numpy(c).to(self.device), torch.from_numpy(s).to(self.device))

    # backend.hpp:26
    def embedding(self, token_id: int, weights, output):
        check(lib().q3_embedding(_p(weights), weights.shape[0], weights.shape[1], token_id, _p(output),
                                 self._stream()))

    # backend.hpp:27
    def matmul(self, input, weights, output):
        check(lib().q3_gemv(_p(input), _p(weights), _p(output), weights.shape[0], weights.shape[1], self._stream()))

    def gemm(self, x, weights, output):
        """Batched matmul of the prefill: output[m, n] = x[m, k] . weights[n, k]^T (q3_gemm)."""
        m, k = x.shape
        n = weights.shape[0]
        check(lib().q3_gemm(_p(x), _p(weights), _p(output), m, n, k, self._stream()))

    def quantize_e4m3(self, weights, q, scale, c0: int = 0, cols: int | None = None):
        """Row-wise E4M3 with power-of-two scales (q3_quantize_e4m3): q[r, :] = E4M3(weights[r, c0:c0+cols] / scale[r])."""
        rows, full = weights.shape
        cols = full - c0 if cols is None else cols
        check(lib().q3_quantize_e4m3(_p(weights), rows, full, c0, cols, _p(q), _p(scale), self._stream()))

    def pack_e4m3(self, q):
        """Row-major E4M3 [n, k] (uint8 tensor) -> the FP8 GEMV's packed layout (q3_pack_e4m3)."""
        torch = _torch()
        n, k = q.shape
        packed = torch.empty(lib().q3_e4m3_packed_bytes(n, k), dtype=torch.uint8, device=q.device)
        check(lib().q3_pack_e4m3(_p(q), n, k, _p(packed), self._stream()))
        return packed

    def gemv_e4m3(self, x, packed, scale, output):
        """output[n] = (W[n, :] . x) * scale[n], W E4M3 in the packed layout of pack_e4m3 (q3_gemv_e4m3)."""
        n, k = output.numel(), x.numel()
        check(lib().q3_gemv_e4m3(_p(x), _p(packed), _p(scale), _p(output), n, k, self._stream()))

    def quantize_nvfp4(self, weights):
        """BF16 [n, k] (device) -> (packed NVFP4 bytes in the GEMV's layout, row scales)
        (q3_quantize_nvfp4)."""
        torch = _torch()
        n, k = weights.shape
        packed = torch.empty(lib().q3_nvfp4_packed_bytes(n, k), dtype=torch.uint8, device=weights.device)
        scale = torch.empty(n, dtype=torch.float32, device=weights.device)
        check(lib().q3_quantize_nvfp4(_p(weights), n, k, _p(packed), _p(scale), self._stream()))
        return packed, scale

    def dequant_nvfp4(self, packed, scale, n: int, k: int):
        """The exact BF16 values [n, k] of a packed NVFP4 matrix (q3_dequant_nvfp4)."""
        torch = _torch()
        out = torch.empty((n, k), dtype=torch.bfloat16, device=packed.device)
        check(lib().q3_dequant_nvfp4(_p(packed), _p(scale), n, k, _p(out), self._stream()))
        return out

    def gemv_nvfp4(self, x, packed, scale, output):
        """output[n] = W[n, :] . x for a packed NVFP4 W (q3_gemv_nvfp4)."""
        n, k = output.numel(), x.numel()
        check(lib().q3_gemv_nvfp4(_p(x), _p(packed), _p(scale), _p(output), n, k, self._stream()))

    # backend.hpp:28
    def rmsnorm(self, input, weight, output, epsilon: float):
        check(lib().q3_rmsnorm(_p(input), _p(weight), _p(output), input.numel(), epsilon, self._stream()))

    # backend.hpp:29
    def rmsnorm_add(self, residual, residual_update, weight, output, epsilon: float):
        check(lib().q3_rmsnorm_add(_p(residual), _p(residual_update), _p(weight), _p(output), residual.numel(),
                                   epsilon, self._stream()))

    # backend.hpp:30
    def rope(self, values, cache: RopeCache, position: int):
        check(lib().q3_rope(_p(values), _p(cache.cosine), _p(cache.sine), values.shape[0], values.shape[1],
                            position, self._stream()))

    # backend.hpp:31; key/value are the reference KV layout [capacity, kv_heads, head_dim]
    def self_attention(self, query, key, value, output, position: int):
        torch = _torch()
        need = lib().q3_attention_workspace_bytes(query.shape[0], key.shape[1], key.shape[0])
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        check(lib().q3_attention(_p(query), _p(key), _p(value), _p(output), query.shape[0], key.shape[1],
                                 query.shape[1], position, _p(self._ws), self._ws.numel(), self._stream()))

    def self_attention_paged(self, query, k_pages, v_pages, page_table, output, position: int):
        torch = _torch()
        need = lib().q3_attention_workspace_bytes(query.shape[0], k_pages.shape[1], position + 1)
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        check(lib().q3_attention_paged(_p(query), _p(k_pages), _p(v_pages), _p(page_table), _p(output),
                                       query.shape[0], k_pages.shape[1], query.shape[1], k_pages.shape[2],
                                       position, _p(self._ws), self._ws.numel(), self._stream()))

    # backend.hpp:32
    def add(self, left, right, output):
        check(lib().q3_add(_p(left), _p(right), _p(output), output.numel(), self._stream()))

    # backend.hpp:33
    def silu(self, gate, up, output):
        check(lib().q3_silu_mul(_p(gate), _p(up), _p(output), output.numel(), self._stream()))

    # backend.hpp:33-34
    def qk_norm_rope(self, query, key, q_norm, k_norm, cache: RopeCache, token_pos: int, eps: float):
        check(lib().q3_qk_norm_rope(_p(query), _p(key), _p(q_norm), _p(k_norm), _p(cache.cosine), _p(cache.sine),
                                    query.shape[0], key.shape[0], query.shape[1], token_pos, eps, self._stream()))

    # ---- bounded paged KV cache (cache.py, q3_cache_*): no counterpart in backend.hpp
    # (checks written for the host time that they cost in every call)

    def _heads(self, name: str, t, n: int, heads: int, index: int) -> int:
        """The row stride of t, a bf16 [n, heads, 128] tensor on device `index` whose rows are contiguous."""
        if t.dtype is self._bf16 and t.shape == (n, heads, 128) and t.get_device() == index:
            row, head, dim = t.stride()
            if dim == 1 and (head == 128 or heads == 1):
                return row if n > 1 else 128 * heads
        raise ValueError(f"{name} must be a bf16 [{n}, {heads}, 128] tensor on {self.device} with contiguous rows")

    def _ints(self, name: str, t, n: int, index: int) -> int:
        if t.dtype is not self._i32 or t.dim() != 1 or t.numel() != n or t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of {n} on {self.device}")
        return t.data_ptr()

    def _cache_call(self, cache):
        """The library, the cache's device index and the current stream there."""
        index = self.device.index
        if cache.device.index != index or not cache.h:
            raise ValueError(f"the cache is closed or on {cache.device}, this backend on {self.device}")
        stream = self._raw_stream(index)
        if stream not in cache._streams:
            cache._used_on(stream)
        return lib(), index, stream

    def cache_append(self, cache, query, key, value, q_norm, k_norm, rope: RopeCache, token_pos, slots, query_out,
                     epsilon: float, lens_out=None, row_seq=None):
        """New tokens into `cache` (q3_cache_append): row i of query / key / value (bf16 [n, heads, 128], rows may
        be strided) is normalised and rotated as qk_norm_rope does at token_pos[i]; the query goes to query_out (may
        be query), key and value to slot slots[i] of sequence row_seq[i] (None: sequence i).  slots[i] = -1 skips
        the row.  lens_out[i] = slots[i] + 1 (may be slots)."""
        L, index, stream = self._cache_call(cache)
        n, qh = query.shape[0], query.shape[1]
        qs = self._heads("query", query, n, qh, index)
        ks = self._heads("key", key, n, cache.kv_heads, index)
        vs = self._heads("value", value, n, cache.kv_heads, index)
        os_ = self._heads("query_out", query_out, n, qh, index)
        cosine, sine = rope.cosine, rope.sine
        for t in (q_norm, k_norm):
            if t.dtype is not self._bf16 or t.numel() != 128 or t.get_device() != index or not t.is_contiguous():
                raise ValueError("q_norm and k_norm must be contiguous bf16 tensors of 128")
        for t in (cosine, sine):
            if (t.dtype is not self._f32 or t.dim() != 2 or t.shape[1] != 64 or t.get_device() != index
                    or not t.is_contiguous()):
                raise ValueError("RoPE tables must be contiguous fp32 [positions, 64]")
        if sine.shape[0] != cosine.shape[0]:
            raise ValueError("RoPE tables differ in length")
        status = L.q3_cache_append(
            cache.h, query.data_ptr(), qs, key.data_ptr(), ks, value.data_ptr(), vs, q_norm.data_ptr(),
            k_norm.data_ptr(), cosine.data_ptr(), sine.data_ptr(), cosine.shape[0],
            self._ints("token_pos", token_pos, n, index), self._ints("slots", slots, n, index),
            None if row_seq is None else self._ints("row_seq", row_seq, n, index), n, qh, query_out.data_ptr(), os_,
            None if lens_out is None else self._ints("lens_out", lens_out, n, index), epsilon, stream)
        if status:
            check(status)

    def cache_attention(self, cache, query, lens, output, accumulate: bool = True):
        """output[r] = attention of query[r] (bf16 [rows, q_heads, 128], rows may be strided) over slots
        0 .. lens[r] - 1 of sequence r (q3_cache_attention); accumulate adds each slot's probabilities, summed over
        the query heads of its kv head, to cache.weights.  output may be query.  An infinite value in a slot below the
        length makes its dimension infinite, or NaN where the formula does."""
        L, index, stream = self._cache_call(cache)
        rows, qh = cache.rows, query.shape[1]
        qs = self._heads("query", query, rows, qh, index)
        os_ = self._heads("output", output, rows, qh, index)
        at = self._ints("lens", lens, rows, index)
        ws = cache._scratch(("attention", qh, accumulate))
        status = L.q3_cache_attention(cache.h, query.data_ptr(), qs, at, output.data_ptr(), os_, qh, accumulate,
                                      ws.data_ptr(), ws.numel(), stream)
        if status:
            check(status)

    def cache_evict(self, cache, lens, next_pos, keep: int, recent: int, lens_out, weights_out=None,
                    positions_out=None):
        """Shrinks every sequence longer than `keep` to `keep` slots per kv head (q3_cache_evict): slots at positions
        >= next_pos[r] - recent first, then the largest weights, the lower slot among equals.  In place, or weights
        and positions to weights_out and positions_out (laid out as the cache's).  lens_out[r] = min(lens[r], keep)
        (may be lens)."""
        L, index, stream = self._cache_call(cache)
        for t, like in ((weights_out, cache.weights), (positions_out, cache.positions)):
            if t is not None and (like is None or t.dtype is not like.dtype or t.shape != like.shape or
                                  t.stride() != like.stride() or t.get_device() != index):
                raise ValueError("weights_out and positions_out must be laid out as the cache's")
        if keep < 1 or recent < 0:
            raise ValueError("cache_evict: keep must be at least 1 and recent at least 0")
        rows = cache.rows
        a, b, c = (self._ints(name, t, rows, index)
                   for name, t in (("lens", lens), ("next_pos", next_pos), ("lens_out", lens_out)))
        ws = cache._scratch(("evict", keep))
        status = L.q3_cache_evict(cache.h, a, b, keep, recent, None if weights_out is None else weights_out.data_ptr(),
                                  None if positions_out is None else positions_out.data_ptr(), c, ws.data_ptr(),
                                  ws.numel(), stream)
        if status:
            check(status)

    # backend.hpp:35 -- synchronises to return the id, as the reference does
    def argmax(self, logits) -> int:
        torch = _torch()
        if self._idx is None:
            self._idx = torch.zeros(1, dtype=torch.int32, device=self.device)
        check(lib().q3_argmax(_p(logits), logits.numel(), _p(self._idx), self._stream()))
        return int(self._idx.item())


def fill_normal(dst, seed: int, tensor_id: int, rows: int, cols: int, row0: int = 0, col0: int = 0,
                full_cols: int | None = None, stream: int = 0):
    check(lib().q3_fill_normal(_p(dst), seed, tensor_id, rows, cols, row0, col0, full_cols or cols, cols, stream))


def prompt_ids(n: int, seed: int = 1, vocab: int = 151936) -> np.ndarray:
    out = np.empty(n, np.uint32)
    lib().q3_prompt_ids(out.ctypes.data, n, seed, vocab)
    return out


def rope_tables(max_pos: int, head_dim: int = 128, theta: float = 1e6):
    c = np.empty((max_pos, head_dim // 2), np.float32)
    s = np.empty_like(c)
    check(lib().q3_rope_tables(max_pos, head_dim, theta, c.ctypes.data, s.ctypes.data))
    return c, s
