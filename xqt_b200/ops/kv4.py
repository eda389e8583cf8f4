"""A paged cache of keys and values in 4 bits, and attention over it.

No counterpart in xqt.  The codes of one token and head go with one scale and one minimum in the activation type (asymmetric, per token and
head), so a key of 128 channels takes 68 bytes where bf16 takes 256.  Layout: ``include/xqt_b200.h``.
"""

from __future__ import annotations

import ctypes

import torch

from .. import native
from ..errors import XQTBackendError
from .rotary import _rows16, _steps

_Strides = ctypes.c_longlong * 4
HEAD_DIMS = (64, 128, 256)
_native = None             # the native call path, once a call has been made


def allocate_kv4_cache(pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device=None):
    """``(codes, params)`` of a cache of ``pages`` pages, zeros: every key and value stands for 0 until it is written."""

    if pages < 0 or kv_heads < 1 or head_dim not in HEAD_DIMS or dtype not in (torch.float16, torch.bfloat16):
        raise XQTBackendError(f"allocate_kv4_cache expects fp16/bf16 and a head dimension of {HEAD_DIMS}")
    if not 16 <= page_size <= 4096 or page_size & (page_size - 1):
        raise XQTBackendError("the page size is a power of two from 16 to 4096")
    codes = torch.zeros((pages, 2, kv_heads, page_size, head_dim // 2), dtype=torch.uint8, device=device)
    return codes, torch.zeros((pages, 2, kv_heads, page_size, 2), dtype=dtype, device=device)


def _cache(what: str, codes: torch.Tensor, params: torch.Tensor) -> tuple[int, int, int, int]:
    """Pages, heads, page size and head dimension of a cache that the kernels take."""

    if codes.ndim != 5 or codes.shape[1] != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous():
        raise XQTBackendError(f"{what}: codes are contiguous uint8 [pages, 2, heads, page_size, dim / 2]")
    pages, _, heads, page_size, half = codes.shape
    if 2 * half not in HEAD_DIMS or heads < 1 or not 16 <= page_size <= 4096 or page_size & (page_size - 1):
        raise XQTBackendError(f"{what}: a head dimension of {HEAD_DIMS} and a page size that is a power of two from 16 to 4096 are served")
    if params.dtype not in (torch.float16, torch.bfloat16) or params.shape != (pages, 2, heads, page_size, 2) or params.device != codes.device \
            or not params.is_contiguous():
        raise XQTBackendError(f"{what}: params are contiguous fp16/bf16 [pages, 2, heads, page_size, 2] on the codes' device")
    if (codes.data_ptr() | params.data_ptr()) % 16:
        raise XQTBackendError(f"{what}: codes and params start on 16 bytes")
    return pages, heads, page_size, 2 * half


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges that two tensors span meet."""

    def span(x: torch.Tensor) -> tuple[int, int]:
        return x.data_ptr(), x.data_ptr() + (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a.numel() > 0 and b.numel() > 0 and a0 < b1 and b0 < a1


def _on_gpu(what: str, codes: torch.Tensor) -> None:
    if not codes.is_cuda:
        raise XQTBackendError(f"{what} expects CUDA tensors")


def _slots(what: str, slots: torch.Tensor, device: torch.device) -> int:
    if slots.ndim != 1 or slots.dtype not in (torch.int32, torch.int64) or slots.device != device or not slots.is_contiguous():
        raise XQTBackendError(f"{what}: slots are contiguous int32/int64 [tokens] on the cache's device")
    return slots.shape[0]


def kv4_append(k: torch.Tensor, v: torch.Tensor, codes: torch.Tensor, params: torch.Tensor, slots: torch.Tensor) -> None:
    """Write the keys and values of ``tokens`` tokens, ``k`` and ``v`` ``[tokens, heads, dim]`` (the type of ``params``, any strides with contiguous
    channels), into the cache.  ``slots[i]`` = ``page * page_size + row`` of token ``i``, distinct in one call; a slot outside the
    cache (-1 for a padded row) is skipped."""

    global _native
    if _native is not None and _native.kv4_append(k, v, codes, params, slots):
        return
    pages, heads, page_size, dim = _cache("kv4_append", codes, params)
    tokens = _slots("kv4_append", slots, codes.device)
    for x in (k, v):
        if x.dtype != params.dtype or x.device != codes.device or x.shape != (tokens, heads, dim):
            raise XQTBackendError("kv4_append: keys and values are [tokens, heads, dim] in the type of params, on the cache's device")
    _on_gpu("kv4_append", codes)
    if not tokens:
        return
    if not _rows16(k):
        k = k.clone(memory_format=torch.contiguous_format)
    if not _rows16(v):
        v = v.clone(memory_format=torch.contiguous_format)
    with torch.cuda.device(codes.device):
        code = native.library().xqt_b200_kv4_append(
            k.data_ptr(), v.data_ptr(), codes.data_ptr(), params.data_ptr(), slots.data_ptr(), _Strides(*_steps(k), *_steps(v)), tokens, heads, dim, pages,
            page_size, slots.dtype == torch.int64, native.DTYPE_CODE[params.dtype], native.stream_handle(codes.device))
    native.check(code, "xqt_b200_kv4_append")
    _native = native.attention_host()


def kv4_gather(codes: torch.Tensor, params: torch.Tensor, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the slots hold, ``[tokens, heads, dim]`` in the type of ``params``; zeros for a slot outside the cache."""

    global _native
    if _native is not None:
        done = _native.kv4_gather(codes, params, slots)
        if done is not None:
            return done
    pages, heads, page_size, dim = _cache("kv4_gather", codes, params)
    tokens = _slots("kv4_gather", slots, codes.device)
    _on_gpu("kv4_gather", codes)
    k = torch.empty((tokens, heads, dim), dtype=params.dtype, device=codes.device)
    v = torch.empty_like(k)
    if tokens:
        with torch.cuda.device(codes.device):
            code = native.library().xqt_b200_kv4_gather(
                codes.data_ptr(), params.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), tokens, heads, dim, pages, page_size,
                slots.dtype == torch.int64, native.DTYPE_CODE[params.dtype], native.stream_handle(codes.device))
        native.check(code, "xqt_b200_kv4_gather")
        _native = native.attention_host()
    return k, v


def kv4_attention(q: torch.Tensor, codes: torch.Tensor, params: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                  query_starts: torch.Tensor | None = None, scale: float | None = None, window: int | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale * q K^T + mask) V`` over the cache, ``[tokens, q_heads, dim]`` like ``q``.

    ``q`` (the type of ``params``, any strides with contiguous channels); consecutive query heads share a key head.  ``block_table`` int32
    ``[batch, width]``: the pages of each sequence; a number outside the cache (-1) is a page whose keys are not seen.  ``seq_lens`` int32
    ``[batch]``: keys of each sequence, its new tokens included.  ``query_starts`` int32 ``[batch + 1]``: sequence ``b`` has the rows
    ``query_starts[b]`` to ``query_starts[b + 1]`` of ``q`` (ascending), which are its last tokens; None: one row per sequence.  A query sees the keys
    up to its own position, with ``window`` the last ``window`` of them.  A row that sees nothing is 0.  ``scale``: ``dim ** -0.5`` by default.

    Lengths stay on the device (the call can be captured in a CUDA graph and replayed with others); they are clamped to the table and to the rows
    of ``q``.  Rows of ``q`` that belong to no sequence are not written: in a new result they hold anything, in ``out`` (contiguous)
    what they held.  ``out`` may be ``q`` itself where that is contiguous, but may not overlap it otherwise.

    The products take fp16 operands under powers of two that neighbours share, also those that a row does not see: in prompts an element of a key keeps its
    precision down to 2^-28 of the largest in its 64 keys, an element of a value down to 2^-28 of the largest in the (up to 16,384) keys up to
    its chunk's end, and counts as 0 below 2^-39; for few queries a probability times the scale of its value does so down to 2^-29 and below 2^-40 of the
    largest such scale so far.  Scores and what they are summed from stay below 2^100.

    Waits inside the kernels are bounded.  Should one run out, that call's result is wrong: the next call on the device raises (:func:`xqt_b200.native.check_waits`
    does so without one, after a synchronisation or a graph's replay)."""

    global _native
    if _native is not None:
        done = _native.kv4_attention(q, codes, params, block_table, seq_lens, query_starts, scale, window, out)
        if done is not None:
            return done
    pages, kv_heads, page_size, dim = _cache("kv4_attention", codes, params)
    device = codes.device
    if q.ndim != 3 or q.dtype != params.dtype or q.device != device or q.shape[2] != dim or q.shape[1] < 1 or q.shape[1] % kv_heads:
        raise XQTBackendError("kv4_attention: queries are [tokens, heads, dim] in the type of params, a multiple of the cache's heads")
    tokens, q_heads, _ = q.shape
    if block_table.ndim != 2 or block_table.dtype != torch.int32 or block_table.device != device or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise XQTBackendError("kv4_attention: the block table is int32 [batch, width] on the cache's device")
    batch, width = block_table.shape
    if seq_lens.ndim != 1 or seq_lens.shape[0] != batch or seq_lens.dtype != torch.int32 or seq_lens.device != device or not seq_lens.is_contiguous():
        raise XQTBackendError("kv4_attention: seq_lens are contiguous int32 [batch] on the cache's device")
    if query_starts is None:
        if tokens != batch:
            raise XQTBackendError("kv4_attention: without query_starts there is one row of queries for each sequence")
    elif query_starts.ndim != 1 or query_starts.shape[0] != batch + 1 or query_starts.dtype != torch.int32 or query_starts.device != device \
            or not query_starts.is_contiguous():
        raise XQTBackendError("kv4_attention: query_starts are contiguous int32 [batch + 1] on the cache's device")
    if window is not None and window < 1:
        raise XQTBackendError("kv4_attention: a window holds a key at least")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) < 2.0 ** 127:          # the kernels hold scale * log2(e) in fp32
        raise XQTBackendError("kv4_attention: the scale is finite and below 2^127")
    _on_gpu("kv4_attention", codes)
    if out is None:
        out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise XQTBackendError("kv4_attention: out has the shape, type and device of the queries, contiguous and on 16 bytes")
    elif _overlap(q, out) and not (q.data_ptr() == out.data_ptr() and q.is_contiguous()):
        raise XQTBackendError("kv4_attention: out is the queries themselves (contiguous) or does not overlap them")
    if tokens and batch:
        if not _rows16(q):
            q = q.clone(memory_format=torch.contiguous_format)
        library = native.library()
        native.check_waits(device)
        with torch.cuda.device(device):
            need = library.xqt_b200_kv4_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, dim, query_starts is not None)
            workspace = torch.empty(need, dtype=torch.uint8, device=device)      # the allocator's: each captured graph has its own
            code = library.xqt_b200_kv4_attention(
                q.data_ptr(), codes.data_ptr(), params.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), native.ptr(query_starts), out.data_ptr(),
                _Strides(*_steps(q), block_table.stride(0), 0), tokens, batch, q_heads, kv_heads, dim, pages, page_size, width,
                0 if window is None else min(int(window), 2 ** 31 - 1), native.DTYPE_CODE[q.dtype], scale, workspace.data_ptr(), need,
                native.pinned_status(device).data_ptr(), native.stream_handle(device))
        native.check(code, "xqt_b200_kv4_attention")
        _native = native.attention_host()
    return out


__all__ = ["HEAD_DIMS", "allocate_kv4_cache", "kv4_append", "kv4_attention", "kv4_gather"]
