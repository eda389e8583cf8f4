"""Outputs of the rotation that would overwrite each other or an input that is still to be read."""

from __future__ import annotations

import pytest
import torch

from conftest import seeded
from xqt_b200.errors import XQTBackendError
from xqt_b200.ops.rotary import qk_norm_rope, rotary_frequencies

pytestmark = pytest.mark.gpu


def test_the_same_memory_twice():
    device = torch.device("cuda", 0)
    x = torch.randn((5, 8, 64), generator=seeded(1)).bfloat16().to(device)
    q, k, positions, frequencies = x[:, :4], x[:, 4:], torch.arange(5, device=device), rotary_frequencies(64, device=device)[0]
    fresh = torch.empty((5, 4, 64), dtype=torch.bfloat16, device=device)
    for out in ((fresh, fresh), (k, fresh), (fresh, q), (k, q)):
        with pytest.raises(XQTBackendError):
            qk_norm_rope(q, k, positions, frequencies, out=out)
    want = qk_norm_rope(q, k, positions, frequencies)
    qk_norm_rope(q, k, positions, frequencies, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
