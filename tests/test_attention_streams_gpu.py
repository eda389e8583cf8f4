"""The forms of attention that keep parts of items in a workspace (the list of few queries, and prompts): on two streams, in two graphs, again and again."""

from __future__ import annotations

import pytest
import torch

from attention_reference import attention
from test_kv4_gpu import DEVICE, _vectors, make_cache, wide
from xqt_b200 import native
from xqt_b200.ops.kv4 import kv4_attention

pytestmark = pytest.mark.gpu

# lengths, queries: single tokens and drafted ones (the wide table takes them to the list, whose items are shared by many CTAs), prompts, and all of them
FORMS = {"tokens": ([3000, 1200, 1, 9000], None), "drafts": ([3000, 12000], [3, 7]), "prompts": ([3000, 1500], [90, 700]), "mixed": ([2000, 5000, 700], [300, 1, 6])}


def arguments(form, dtype, dim, heads=2, seed=95):
    lens, counts = FORMS[form]
    codes, params, table = make_cache(lens, heads, dim, 64, dtype, seed)
    starts = None if counts is None else torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32, device=DEVICE)
    rows = len(lens) if counts is None else sum(counts)
    return lens, rows, (codes, params, wide(table, 64), torch.tensor(lens, dtype=torch.int32, device=DEVICE)), starts


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 128), (torch.bfloat16, 64), (torch.bfloat16, 256)])
@pytest.mark.parametrize("form", FORMS)
def test_two_streams_and_two_captured_graphs(form, dtype, dim):
    lens, rows, cache, starts = arguments(form, dtype, dim)
    qs = [_vectors(rows, 8, dim, dtype, 96 + i).to(DEVICE) for i in range(2)]
    want = [kv4_attention(q, *cache, query_starts=starts) for q in qs]
    assert not torch.equal(*want)
    graphs, held = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(kv4_attention(q, *cache, query_starts=starts))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(30):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    got = [[], []]
    for _ in range(30):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(kv4_attention(qs[i], *cache, query_starts=starts))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    cache[3].sub_(1)                                    # lengths live on the device, for both graphs
    for graph in graphs:
        graph.replay()
    again = [kv4_attention(q, *cache, query_starts=starts) for q in qs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, again)) and native.workspace_status(DEVICE) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_same_bits_every_time(form, dim, dtype):
    lens, rows, cache, starts = arguments(form, dtype, dim, heads=4)
    q = _vectors(rows, 16, dim, dtype, 98).to(DEVICE)
    first = kv4_attention(q, *cache, query_starts=starts)
    for _ in range(10):
        assert torch.equal(kv4_attention(q, *cache, query_starts=starts), first)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,lens,counts", [(128, [3000], [70]), (64, [700, 2000, 64], [65, 300, 9]), (256, [100] * 10, [60] * 10)])
def test_many_rows_in_the_kernel_of_few_queries(dtype, dim, lens, counts):
    """Calls of so little work that all their sequences stay with that kernel are held to its own bound: one rounding besides the result's."""
    codes, params, table = make_cache(lens, 2, dim, 64, dtype, 99)
    assert sum(counts) * 8 * table.shape[1] * 64 * dim <= 768e6              # the rule between the kernels
    q = _vectors(sum(counts), 8, dim, dtype, 100)
    seq_lens, starts = (torch.tensor(x, dtype=torch.int32) for x in (lens, [sum(counts[:b]) for b in range(len(counts) + 1)]))
    got = kv4_attention(q.to(DEVICE), codes, params, table, seq_lens.to(DEVICE), query_starts=starts.to(DEVICE)).double()
    want, bound = attention(q.to(DEVICE), codes, params, table, seq_lens, starts)
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), f"{float(over.max())} over a bound of {float(bound.max())}"


def test_few_rows_beside_prompts_keep_the_tighter_bound():
    """In one call with prompts the sequences of at most 32 rows go to the kernel for few queries: their rows are held to its bound."""
    lens, counts = [40, 700, 33, 512, 2000, 900], [8, 300, 1, 40, 700, 2]
    codes, params, table = make_cache(lens, 2, 128, 32, torch.float16, 101)
    q = _vectors(sum(counts), 8, 128, torch.float16, 102)
    seq_lens, starts = (torch.tensor(x, dtype=torch.int32) for x in (lens, [sum(counts[:b]) for b in range(len(counts) + 1)]))
    got = kv4_attention(q.to(DEVICE), codes, params, wide(table, 32), seq_lens.to(DEVICE), query_starts=starts.to(DEVICE)).double()
    want, tight = attention(q.to(DEVICE), codes, params, table, seq_lens, starts)
    loose = attention(q.to(DEVICE), codes, params, table, seq_lens, starts, rounded=torch.float16)[1]
    few = torch.repeat_interleave(torch.tensor(counts) * 4 <= 32, torch.tensor(counts)).to(DEVICE)
    assert bool(((got - want).abs()[few] <= tight[few]).all()) and bool(((got - want).abs() <= loose).all())
