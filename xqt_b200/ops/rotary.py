"""Norms of query and key heads with the position rotation, in one pass over the output of a QKV projection.

No counterpart in xqt, whose operators end at the quantised projections.  The rotation takes positions with one axis (text) or
several (time, height, width of pictures and video), a ladder of frequencies per axis or one ladder whose pairs are shared out
among the axes: every pair of channels has a frequency and an axis of its own.
"""

from __future__ import annotations

import ctypes
import math

import torch

from .. import native
from ..errors import XQTBackendError

_Strides = ctypes.c_longlong * 10
_native = None             # the native call path, once a call has been made


def rotary_frequencies(rotary_dim: int, *, theta: float = 10000.0, sections=None, ladders=None, device=None):
    """``(frequencies, axes)`` of the pairs of ``rotary_dim`` channels, as :func:`qk_norm_rope` takes them.

    With neither option one axis and the ladder ``theta ** (-2j / rotary_dim)`` (``axes`` is None).  ``sections``: the same
    ladder, whose first ``sections[0]`` pairs follow axis 0, the next ``sections[1]`` axis 1, and so on.  ``ladders``: axis ``i`` has
    ``ladders[i]`` channels with a ladder of its own, ``theta ** (-2j / ladders[i])``."""

    if rotary_dim < 2 or rotary_dim % 2 or (sections is not None and ladders is not None):
        raise XQTBackendError("rotary_frequencies expects an even number of channels and at most one of sections and ladders")
    if not (math.isfinite(theta) and theta > 0):
        raise XQTBackendError("rotary_frequencies expects a positive theta")
    pairs = rotary_dim // 2
    if ladders is not None:
        if any(n < 2 or n % 2 for n in ladders) or sum(ladders) != rotary_dim:
            raise XQTBackendError("ladders are even numbers of channels that add up to rotary_dim")
        values = [theta ** (-2 * j / n) for n in ladders for j in range(n // 2)]
        owner = [i for i, n in enumerate(ladders) for _ in range(n // 2)]
    else:
        values = [theta ** (-j / pairs) for j in range(pairs)]
        owner = None
        if sections is not None:
            if any(n < 0 for n in sections) or sum(sections) != pairs:
                raise XQTBackendError("sections are numbers of pairs that add up to rotary_dim / 2")
            owner = [i for i, n in enumerate(sections) for _ in range(n)]
    frequencies = torch.tensor(values, dtype=torch.float64, device=device)
    return frequencies, None if owner is None else torch.tensor(owner, dtype=torch.int32, device=device)


def _dense(shape: tuple, strides: tuple) -> bool:
    """Whether no two elements of a ``[tokens, heads, dim]`` view share an address."""

    (t, h, d), (st, sh, sd) = shape, strides
    if sd != 1:
        return False
    by_head = (h == 1 or sh >= d) and (t == 1 or st >= (h - 1) * sh + d)
    by_token = (t == 1 or st >= d) and (h == 1 or sh >= (t - 1) * st + d)
    return by_head or by_token


def _rows16(x: torch.Tensor) -> bool:
    """Whether every run of channels starts on 16 bytes."""

    st, sh, sd = x.stride()
    return sd == 1 and x.data_ptr() % 16 == 0 and (st % 8 == 0 or x.shape[0] == 1) and (sh % 8 == 0 or x.shape[1] == 1)


def _steps(x: torch.Tensor) -> tuple[int, int]:
    """Token and head stride, 0 where there is only one."""

    st, sh, _ = x.stride()
    return (st if x.shape[0] > 1 else 0), (sh if x.shape[1] > 1 else 0)


def _bad(message: str):
    raise XQTBackendError(f"qk_norm_rope: {message}")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, *, axes: torch.Tensor | None = None,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False, out=None):
    """RMS norm of each head of ``q`` and ``k`` and their rotation: ``-> (q_out, k_out)``.

    ``q`` ``[tokens, q_heads, dim]``, ``k`` ``[tokens, k_heads, dim]`` (or None): fp16 or bf16, any strides with contiguous channels, as
    slices of a fused projection are; ``dim`` a multiple of 16 up to 256.  ``q_weight`` / ``k_weight`` ``[dim]`` (fp16, bf16 or fp32): the norm
    ``x * rsqrt(mean(x^2) + eps) * weight``; without one that side is not normed.  ``positions`` int32 / int64 ``[tokens]`` or ``[axes, tokens]``;
    ``frequencies`` float64 ``[pairs]``, radians per position of each pair of channels (a multiple of 8 pairs, none: no rotation); ``axes`` int32
    ``[pairs]``, the axis that each pair follows (None: axis 0; numbers outside are clamped).  Pair ``j`` is channels ``(j, j + pairs)``, or
    ``(2j, 2j + 1)`` with ``interleaved``; channels from ``2 * pairs`` on are not turned.  fp32 arithmetic, rounded once; angles are
    off by at most 2^-53 of a turn per position besides (1.5e-6 radians at position 2^31).

    ``out = (q_out, k_out)``: written instead of new tensors; either may be the input itself (in place), but may not overlap an input otherwise, nor may
    they overlap each other."""

    global _native
    if _native is not None and out is None:
        done = _native(q, k, positions, frequencies, axes, q_weight, k_weight, eps, interleaved)
        if done is not None:
            return done
    if q.ndim != 3 or q.dtype not in (torch.float16, torch.bfloat16):
        _bad("expects fp16/bf16 queries [tokens, heads, dim]")
    device, dtype = q.device, q.dtype
    tokens, q_heads, dim = q.shape
    if dim % 16 or not 16 <= dim <= 256 or q_heads < 1:
        _bad("the head dimension is a multiple of 16 up to 256, and there is a head")
    k_heads = 0
    if k is not None:
        if k.ndim != 3 or k.dtype != dtype or k.device != device or k.shape[0] != tokens or k.shape[2] != dim or k.shape[1] < 1:
            _bad("keys are of the queries' type, device, tokens and head dimension")
        k_heads = k.shape[1]
    elif k_weight is not None:
        _bad("a weight for keys, but no keys")
    if frequencies.ndim != 1 or frequencies.dtype != torch.float64 or frequencies.device != device or not frequencies.is_contiguous():
        _bad("expects contiguous float64 frequencies [pairs] on the queries' device")
    pairs = frequencies.shape[0]
    if pairs % 8 or 2 * pairs > dim:
        _bad("the rotated pairs are a multiple of 8 and fit the head dimension")
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != device or positions.ndim not in (1, 2) or positions.shape[-1] != tokens:
        _bad("expects int32/int64 positions [tokens] or [axes, tokens] on the queries' device")
    axis_count = 1 if positions.ndim == 1 else positions.shape[0]
    if axis_count < 1:
        _bad("positions have an axis at least")
    if axes is not None and (axes.ndim != 1 or axes.dtype != torch.int32 or axes.device != device or axes.shape[0] != pairs or not axes.is_contiguous()):
        _bad("axes are contiguous int32 [pairs] on the queries' device")
    weight_dtype = None
    for weight in (q_weight, k_weight):
        if weight is not None:
            if weight.ndim != 1 or weight.shape[0] != dim or weight.device != device or weight.dtype not in native.DTYPE_CODE or not weight.is_contiguous() \
                    or weight_dtype not in (None, weight.dtype):
                _bad("norm weights are contiguous [dim] tensors of one type (fp16, bf16 or fp32) on the queries' device")
            weight_dtype = weight.dtype
    if not q.is_cuda:
        _bad("expects CUDA tensors")
    if out is None:
        q_out = torch.empty((tokens, q_heads, dim), dtype=dtype, device=device)
        k_out = None if k is None else torch.empty((tokens, k_heads, dim), dtype=dtype, device=device)
    else:
        q_out, k_out = out
        for given, x in ((q_out, q), (k_out, k)):
            if (given is None) != (x is None):
                _bad("outputs go with inputs: (q_out, k_out)")
            if given is not None and (given.dtype != dtype or given.device != device or given.shape != x.shape or not _rows16(given)
                                      or not _dense(given.shape, given.stride())):
                _bad("an output has its input's shape, type and device, contiguous channels on 16 bytes, and no shared addresses")
        if tokens and k is not None:
            for a, b in ((q_out, k_out), (q_out, k), (k_out, q)):
                if a.data_ptr() == b.data_ptr():
                    _bad("the outputs do not overlap each other or the other one's input")
    if tokens:
        if not _rows16(q):
            q = q.clone(memory_format=torch.contiguous_format)
        if k is not None and not _rows16(k):
            k = k.clone(memory_format=torch.contiguous_format)
        p = positions.stride()
        strides = _Strides(*_steps(q), *_steps(q_out), *((0, 0, 0, 0) if k is None else (*_steps(k), *_steps(k_out))), p[0] if len(p) == 2 else 0, p[-1])
        with torch.cuda.device(device):
            code = native.library().xqt_b200_qk_norm_rope(
                q.data_ptr(), native.ptr(k), q_out.data_ptr(), native.ptr(k_out), native.ptr(q_weight), native.ptr(k_weight), positions.data_ptr(),
                frequencies.data_ptr(), native.ptr(axes), strides, tokens, q_heads, k_heads, dim, 2 * pairs, axis_count,
                positions.dtype == torch.int64, bool(interleaved), native.DTYPE_CODE[dtype], native.DTYPE_CODE[weight_dtype or torch.float32], float(eps),
                native.stream_handle(device))
        native.check(code, "xqt_b200_qk_norm_rope")
        _native = native.attention_host().qk_norm_rope
    return q_out, k_out


__all__ = ["qk_norm_rope", "rotary_frequencies"]
