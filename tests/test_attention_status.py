"""A wait that ran out inside an attention kernel is reported by the next call.  The kernels' waits do not run out in a test: the word that they write is
set here."""

from __future__ import annotations

import pytest
import torch

from xqt_b200 import native
from xqt_b200.errors import XQTBackendError
from xqt_b200.ops import kv4


def test_reported_once(monkeypatch):
    word = torch.zeros(16, dtype=torch.int32)
    device = torch.device("cuda", 3)
    monkeypatch.setattr(native, "_pinned_status", {3: word})
    native.check_waits(device)
    word[0] = 1
    with pytest.raises(XQTBackendError, match="ran out"):
        native.check_waits(device)
    native.check_waits(device)
    native.check_waits(torch.device("cuda", 4))         # another device's calls are not concerned


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["native", "python"])
@pytest.mark.parametrize("queries", [1, 70])
def test_the_next_call_raises(path, queries):
    device = torch.device("cuda", 0)
    codes, params = kv4.allocate_kv4_cache(64, 1, 64, device=device)
    kv4.kv4_append(*[torch.randn((100, 1, 64), device=device).bfloat16() for _ in range(2)], codes, params, torch.arange(100, device=device))
    q = torch.randn((queries, 2, 64), device=device).bfloat16()
    table = torch.arange(64, dtype=torch.int32, device=device).repeat(1, 300)          # so wide that many queries go to the prompt kernel
    lens, starts = torch.tensor([100], dtype=torch.int32, device=device), torch.tensor([0, queries], dtype=torch.int32, device=device)

    def call():
        if path == "python":
            kv4._native = None
        return kv4.kv4_attention(q, codes, params, table, lens, query_starts=starts)

    first = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    word = native.pinned_status(device)
    assert word.is_pinned() and native.workspace_status(device) == 0
    word[0] = 1
    assert native.workspace_status(device) == 1
    with pytest.raises(XQTBackendError, match="ran out"):
        call()
    assert native.workspace_status(device) == 0 and torch.equal(call(), first)
    graph.replay()
    torch.cuda.synchronize()
    native.check_waits(device)
    assert torch.equal(held, first)
