"""Where the attention over the 4-bit cache may write."""

from __future__ import annotations

import pytest
import torch

from test_kv4_gpu import DEVICE, _vectors, make_cache, wide
from xqt_b200.errors import XQTBackendError
from xqt_b200.ops import kv4

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def attention(request):
    def call(*args, **options):
        if request.param == "python":
            kv4._native = None
        return kv4.kv4_attention(*args, **options)

    return call


def test_out_that_overlaps_the_queries_is_refused(attention):
    lens = [40, 90]
    codes, params, table = make_cache(lens, 2, 64, 16, torch.float16, 91)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    buffer = _vectors(4, 8, 64, torch.float16, 92).to(DEVICE)
    q = buffer[:2, :4].clone()
    attention(q, codes, params, table, seq_lens)
    flat = buffer.view(-1)
    for bad_q, bad_out in ((buffer[:2, :4], flat[:512].view(2, 4, 64)),                       # slices of one buffer, written over by contiguous rows
                           (flat[:512].view(2, 4, 64), flat[64:576].view(2, 4, 64)),          # one head further
                           (flat[:512].view(4, 2, 64).transpose(0, 1), flat[:512].view(2, 4, 64))):
        with pytest.raises(XQTBackendError, match="overlap"):
            attention(bad_q, codes, params, table, seq_lens, out=bad_out)
    out = flat[1024:1536].view(2, 4, 64)              # beside them in the same buffer
    attention(buffer[:2, :4], codes, params, table, seq_lens, out=out)
    assert torch.equal(out, attention(buffer[:2, :4].contiguous(), codes, params, table, seq_lens))


@pytest.mark.parametrize("lens,counts,broad", [([40, 900, 1], None, False), ([40, 9000, 1], None, True), ([700, 300], [5, 2], False), ([900, 300, 2000], [300, 20, 700], True)])
def test_in_place(attention, lens, counts, broad):
    """The clusters, the list, drafted tokens and prompts (with items that several CTAs share) read all of a row's queries before they write it."""
    codes, params, table = make_cache(lens, 2, 128, 64, torch.bfloat16, 93)
    table = wide(table, 64) if broad else table
    q = _vectors(len(lens) if counts is None else sum(counts), 8, 128, torch.bfloat16, 94).to(DEVICE)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    starts = None if counts is None else torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32, device=DEVICE)
    want = attention(q, codes, params, table, seq_lens, query_starts=starts)
    for _ in range(3):
        x = q.clone()
        assert attention(x, codes, params, table, seq_lens, query_starts=starts, out=x).data_ptr() == x.data_ptr() and torch.equal(x, want)
