"""Calls of the attention operators that are refused because the kernels cannot hold them: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from xqt_b200 import native
from xqt_b200.errors import XQTBackendError
from xqt_b200.ops.kv4 import allocate_kv4_cache, kv4_attention


@pytest.mark.parametrize("scale", [2.0 ** 127, -3e38, 1e300, float("inf")])
def test_scales_beyond_fp32(scale):
    """Finite in 64 bits, but scale * log2(e) is not in the 32 that the kernels multiply by: every score would be infinite or NaN."""
    codes, params = allocate_kv4_cache(1, 2, 64, page_size=16, dtype=torch.float16)
    with pytest.raises(XQTBackendError, match="scale"):
        kv4_attention(torch.zeros(1, 4, 64, dtype=torch.float16), codes, params, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), scale=scale)
    entry = lambda value, tokens: native.library().xqt_b200_kv4_attention(  # noqa: E731
        16, 16, 16, 16, 16, 0, 16, (ctypes.c_longlong * 4)(), tokens, 1, 1, 1, 64, 1, 16, 1, 0, 0, value, 0, 0, 0, 0)
    assert entry(scale, 0) == 1 and entry(-1.7e38, 0) == 0        # no tokens: nothing to launch


def test_address_ranges():
    from xqt_b200.ops.kv4 import _overlap

    x = torch.empty(4 * 6 * 64)
    y = x.view(4, 6, 64)
    assert _overlap(y, y) and _overlap(y[:, :3], y[:, 3:]) and not _overlap(y[:2], y[2:]) and not _overlap(y[:1, :3], y[:1, 3:])
    assert _overlap(y[:2], y[1:]) and not _overlap(y[:0], y) and not _overlap(y, torch.empty(1))
