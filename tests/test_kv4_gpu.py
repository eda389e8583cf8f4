"""The 4-bit paged cache and attention over it, against the definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

from attention_reference import attention, pack, quantize, values
from conftest import seeded
from xqt_b200 import native
from xqt_b200.errors import XQTBackendError
from xqt_b200.ops.kv4 import allocate_kv4_cache, kv4_append, kv4_attention, kv4_gather

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
NAN, INF = float("nan"), float("inf")


def _vectors(tokens, heads, dim, dtype, seed, size=1.0):
    return (torch.randn((tokens, heads, dim), generator=seeded(seed)) * size).to(dtype)


# ---------------------------------------------------------------- writing and reading

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 64, 16), (5, 3, 128, 32), (67, 2, 256, 16), (1000, 8, 128, 64), (31, 5, 64, 4096)])
def test_append_and_gather(dtype, wide, tokens, heads, dim, page):
    pages = tokens // page + 3
    k, v = _vectors(tokens, heads, dim, dtype, 1), _vectors(tokens, heads, dim, dtype, 2, 30.0)
    v[0, 0] = 3.0                                     # a constant vector: scale 1, codes 0
    codes, params = allocate_kv4_cache(pages, heads, dim, page_size=page, dtype=dtype, device=DEVICE)
    codes.fill_(0xA5)
    slots = torch.randperm(pages * page, generator=seeded(3))[:tokens].to(wide)
    want_codes, want_params = codes.cpu(), params.cpu()
    for i, x in enumerate((k, v)):
        c, s, m = quantize(x)
        want_codes[slots.long() // page, i, :, slots.long() % page] = pack(c)
        want_params[slots.long() // page, i, :, slots.long() % page] = torch.stack((s, m), -1)
    kv4_append(k.to(DEVICE), v.to(DEVICE), codes, params, slots.to(DEVICE))
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(params.cpu(), want_params)
    got = kv4_gather(codes, params, slots.to(DEVICE))
    for i in (0, 1):
        held = values(want_codes[slots.long() // page, i, :, slots.long() % page], want_params[slots.long() // page, i, :, slots.long() % page])
        # code * scale is exact in fp32, so the sum is rounded once to fp32 and once to the type
        assert torch.equal(got[i].cpu(), held.float().to(dtype))


def test_append_of_strided_vectors_and_padded_rows():
    fused = _vectors(9, 2 + 2 * 2, 128, torch.bfloat16, 4).to(DEVICE)
    codes, params = allocate_kv4_cache(2, 2, 128, page_size=16, device=DEVICE)
    other = [t.clone() for t in (codes, params)]
    slots = torch.tensor([3, -1, 31, 32, 0, 7, -5, 1 << 40, 30], device=DEVICE)
    keep = torch.tensor([0, 2, 4, 5, 8], device=DEVICE)
    k, v = fused[:, 2:4], fused[:, 4:]
    kv4_append(k, v, codes, params, slots)
    kv4_append(k[keep].contiguous(), v[keep].contiguous(), *other, slots[keep])
    assert torch.equal(codes, other[0]) and torch.equal(params, other[1])
    shifted = torch.empty((9, 2, 131), dtype=torch.bfloat16, device=DEVICE)[:, :, 1:129]
    shifted.copy_(k)
    again = [torch.zeros_like(t) for t in (codes, params)]
    kv4_append(shifted, v, *again, slots)
    assert torch.equal(codes, again[0]) and torch.equal(params, again[1])
    got = kv4_gather(codes, params, slots)
    assert all(bool((x[[1, 3, 6, 7]] == 0).all()) for x in got) and bool((got[0][0] != 0).any())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [1, 3, 7])
def test_append_at_every_magnitude_and_on_half_codes(dtype, heads):
    """Ranges from the smallest number of the type to its largest, and vectors that stand exactly between two codes."""
    info = torch.finfo(dtype)
    low, high = (-24, 11) if dtype == torch.float16 else (-133, 122)
    grid = torch.cat([torch.tensor([0.0, 30.0]), torch.randint(0, 31, (62,), generator=seeded(41)).float()])     # scale 2: odd ones are halves
    rows = []
    for e in range(low, high + 1):
        rows += [grid.double() * 2.0 ** e, (grid.double() - 13) * 2.0 ** e, torch.randn(64, generator=seeded(900 + e), dtype=torch.float64) * 2.0 ** e]
    x = torch.stack(rows).clamp(-info.max, info.max).to(dtype)
    x = x[: len(x) // heads * heads].reshape(-1, heads, 64)
    tokens = len(x)
    codes, params = allocate_kv4_cache(tokens // 16 + 1, heads, 64, page_size=16, dtype=dtype, device=DEVICE)
    slots = torch.arange(tokens)
    kv4_append(x.to(DEVICE), x.flip(0).to(DEVICE), codes, params, slots.to(DEVICE))
    for i, y in enumerate((x, x.flip(0))):
        c, s, m = quantize(y)
        assert torch.equal(params.cpu()[slots // 16, i, :, slots % 16], torch.stack((s, m), -1))
        assert torch.equal(codes.cpu()[slots // 16, i, :, slots % 16], pack(c))


def test_vectors_that_are_not_finite():
    x = _vectors(5, 1, 64, torch.bfloat16, 5)
    x[1, 0, 3], x[2, 0, 9], x[3, 0, 0] = NAN, INF, -INF
    x[4, 0, 0], x[4, 0, 1] = 3.3e38, -3.3e38           # the range overflows
    codes, params = allocate_kv4_cache(1, 1, 64, page_size=16, device=DEVICE)
    codes.fill_(255)
    kv4_append(x.to(DEVICE), x.to(DEVICE), codes, params, torch.arange(5, device=DEVICE))
    c, s, m = quantize(x)
    assert torch.equal(codes[0, 0, 0, :5].cpu(), pack(c)[:, 0]) and bool((codes[0, :, 0, 1:5] == 0).all())
    assert bool(torch.isnan(params[0, :, 0, 1:5]).all()) and torch.equal(params[0, 1, 0, 0].cpu(), torch.stack((s, m), -1)[0, 0])
    assert bool(torch.isnan(kv4_gather(codes, params, torch.arange(1, 5, device=DEVICE))[1]).all())


def test_nothing_to_append():
    codes, params = allocate_kv4_cache(1, 2, 64, page_size=16, device=DEVICE)
    empty = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=DEVICE)
    kv4_append(empty, empty, codes, params, torch.empty(0, dtype=torch.int64, device=DEVICE))
    assert kv4_gather(codes, params, torch.empty(0, dtype=torch.int32, device=DEVICE))[0].shape == (0, 2, 64)
    none = allocate_kv4_cache(0, 2, 64, page_size=16, device=DEVICE)
    kv4_append(torch.ones((1, 2, 64), dtype=torch.bfloat16, device=DEVICE), torch.ones((1, 2, 64), dtype=torch.bfloat16, device=DEVICE), *none,
               torch.zeros(1, dtype=torch.int64, device=DEVICE))
    assert bool((kv4_gather(*none, torch.zeros(1, dtype=torch.int64, device=DEVICE))[0] == 0).all())


# ---------------------------------------------------------------- attention

def make_cache(lens, heads, dim, page, dtype, seed, spare=2, size=1.0):
    """A cache whose pages hold random vectors in random order, unused rows NaN, and its table."""

    per = [-(-n // page) for n in lens]
    pages = sum(per) + spare
    gen = seeded(seed)
    x = (torch.randn((pages, 2, heads, page, dim), generator=gen) * size).to(dtype)
    c, s, m = quantize(x)
    codes, params = pack(c), torch.stack((s, m), -1)
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(max(per, default=0), 1) + 1), -1, dtype=torch.int32)
    at, unused = 0, torch.ones(pages, page, dtype=torch.bool)
    for b, n in enumerate(per):
        ids = order[at:at + n]
        table[b, :n] = ids
        at += n
        for i, p in enumerate(ids.tolist()):
            unused[p, :min(page, lens[b] - i * page)] = False
    params.permute(0, 3, 1, 2, 4)[unused] = NAN
    return codes.to(DEVICE), params.to(DEVICE), table.to(DEVICE)


def check(q, codes, params, table, lens, counts=None, **options):
    seq_lens = torch.tensor(lens, dtype=torch.int32)
    starts = None if counts is None else torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32)
    got = kv4_attention(q.to(DEVICE), codes, params, table, seq_lens.to(DEVICE), query_starts=None if starts is None else starts.to(DEVICE), **options)
    # sequences of more than 32 rows for a key head may go to the kernel that forms keys, values and probabilities in fp16
    many = counts is not None and max(counts) * q.shape[1] // codes.shape[2] > 32
    want, bound = attention(q.to(DEVICE), codes, params, table, seq_lens, starts, rounded=torch.float16 if many else None, **options)
    got = got.double()
    rows = ~torch.isnan(want).all(-1).all(-1)
    assert bool(torch.isfinite(got[rows]).all())
    over = (got - want).abs()[rows] - bound[rows]
    assert bool((over <= 0).all()), f"{float(over.max())} over a bound of {float(bound[rows].max())}"
    assert native.workspace_status(DEVICE) == 0
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,each,dim,page", [(1, 1, 64, 16), (2, 4, 128, 64), (8, 4, 128, 16), (2, 8, 64, 32), (1, 16, 128, 128), (3, 5, 128, 32),
                                                 (2, 7, 256, 64), (1, 12, 256, 16), (1, 33, 64, 64)])
@pytest.mark.parametrize("lens", [[1], [0, 2, 17, 64, 65, 300], [777]])
def test_single_tokens(dtype, heads, each, dim, page, lens):
    codes, params, table = make_cache(lens, heads, dim, page, dtype, 11)
    check(_vectors(len(lens), heads * each, dim, dtype, 12), codes, params, table, lens)


@pytest.mark.parametrize("lens,heads,each,dim,page", [([20000], 1, 4, 128, 64), ([4096, 1, 9000, 0, 513], 2, 8, 64, 16), ([5000, 3001], 2, 1, 256, 128)])
def test_long_contexts_split_over_the_gpu(lens, heads, each, dim, page):
    codes, params, table = make_cache(lens, heads, dim, page, torch.bfloat16, 13)
    check(_vectors(len(lens), heads * each, dim, torch.bfloat16, 14), codes, params, table, lens)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,each,dim,page", [(2, 4, 128, 64), (1, 3, 64, 16), (1, 2, 256, 32), (2, 1, 128, 16)])
@pytest.mark.parametrize("window", [None, 1, 33, 100])
def test_a_few_queries_of_each_sequence(dtype, heads, each, dim, page, window):
    lens, counts = [5, 40, 300, 129, 7], [5, 3, 7, 0, 1]
    codes, params, table = make_cache(lens, heads, dim, page, dtype, 15)
    check(_vectors(sum(counts), heads * each, dim, dtype, 16), codes, params, table, lens, counts, window=window)


def test_more_queries_than_keys_and_other_scale():
    lens, counts = [3, 0, 40], [6, 2, 41]
    codes, params, table = make_cache(lens, 2, 64, 16, torch.float16, 17)
    got = check(_vectors(sum(counts), 4, 64, torch.float16, 18), codes, params, table, lens, counts, scale=0.3)
    assert bool((got[:3] == 0).all()) and bool((got[6:9] == 0).all()) and bool((got[3:6] != 0).any())


@pytest.mark.parametrize("window", [1, 63, 64, 1000, 2 ** 31 - 1])
def test_window_of_single_tokens(window):
    lens = [1, 63, 64, 65, 2000]
    codes, params, table = make_cache(lens, 2, 128, 32, torch.bfloat16, 19)
    check(_vectors(5, 8, 128, torch.bfloat16, 20), codes, params, table, lens, window=window)


def test_large_values_and_sharp_rows():
    """Scores far apart (one key takes all), values of very different scales, tiny and huge queries."""

    lens = [500, 500, 500]
    codes, params, table = make_cache(lens, 2, 128, 64, torch.bfloat16, 21, size=4.0)
    params[:, 1, :, ::7] *= 1e-4
    params[:, 1, :, 3::7] *= 1e4
    q = _vectors(3, 8, 128, torch.bfloat16, 22)
    q[0] *= 50
    q[1] *= 1e-6
    q[2, 3] = 0
    check(q, codes, params, table, lens)


def test_zero_and_negative_scales_are_arithmetic():
    lens = [130]
    codes, params, table = make_cache(lens, 1, 64, 16, torch.float16, 23)
    params[:, 1, :, ::3, 0] = 0
    params[:, 1, :, 1::3, 0] *= -1
    q = _vectors(1, 2, 64, torch.float16, 24)
    check(q, codes, params, table, lens)


def test_empty_cache_reads_zeros():
    codes, params = allocate_kv4_cache(3, 2, 64, page_size=16, device=DEVICE)
    table = torch.arange(2, dtype=torch.int32, device=DEVICE).reshape(1, 2)
    got = kv4_attention(_vectors(1, 2, 64, torch.bfloat16, 25).to(DEVICE), codes, params, table, torch.tensor([20], dtype=torch.int32, device=DEVICE))
    assert bool((got == 0).all())


def test_pages_that_are_not_there():
    """Numbers outside the cache hide their keys; lengths past the table and starts outside the rows are cut."""

    lens = [100, 200, 64]
    codes, params, table = make_cache(lens, 2, 128, 16, torch.float16, 26)
    table[0, 2], table[1, 0], table[1, 5] = -1, codes.shape[0], 2 ** 31 - 1
    table[2] = -7
    got = check(_vectors(3, 4, 128, torch.float16, 27), codes, params, table, lens)
    assert bool((got[2] == 0).all())
    check(_vectors(3, 4, 128, torch.float16, 28), codes, params, table, [100, 10 ** 9, -5])
    q = _vectors(6, 4, 128, torch.float16, 29)
    starts = torch.tensor([-3, 2, 1, 99], dtype=torch.int32, device=DEVICE)         # clamped: rows 0-1, none, 1-5 (not ascending: row 1 is anyone's)
    out = kv4_attention(q.to(DEVICE), codes, params, table, torch.tensor([100, 200, 64], dtype=torch.int32, device=DEVICE), query_starts=starts)
    assert bool((out[2:] == 0).all()) and bool((out[0] != 0).any())        # the third sequence's pages are none


def test_rows_of_no_sequence_stay():
    lens = [50, 20]
    codes, params, table = make_cache(lens, 1, 64, 16, torch.bfloat16, 30)
    q = _vectors(9, 2, 64, torch.bfloat16, 31).to(DEVICE)
    out = torch.full_like(q, 7.0)
    starts = torch.tensor([2, 4, 5], dtype=torch.int32, device=DEVICE)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    got = kv4_attention(q, codes, params, table, seq_lens, query_starts=starts, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[:2] == 7).all()) and bool((out[5:] == 7).all()) and not bool((out[2:5] == 7).any())
    first = kv4_attention(q[2:5], codes, params, table, seq_lens, query_starts=starts - 2)
    assert torch.equal(first, out[2:5])


@pytest.mark.parametrize("counts", [None, [3, 2]])
def test_infinities_and_nan_in_hidden_places(counts):
    lens = [70, 90]
    codes, params, table = make_cache(lens, 1, 128, 16, torch.bfloat16, 32)
    q = _vectors(2 if counts is None else 5, 4, 128, torch.bfloat16, 33)
    if counts is not None:      # the last key of sequence 0 is NaN, its values infinite: only its last query sees them
        page, row = int(table[0, 69 // 16]), 69 % 16
        params[page, 0, 0, row] = NAN
        params[page, 1, 0, row] = INF
        clean = [t.clone() for t in (codes, params)]
        clean[1][page, :, 0, row] = 1.0
        seq_lens, starts = (torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in (lens, [0, 3, 5]))
        got = kv4_attention(q.to(DEVICE), codes, params, table, seq_lens, query_starts=starts)
        want = kv4_attention(q.to(DEVICE), *clean, table, seq_lens, query_starts=starts)
        keep = [0, 1, 3, 4]
        assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[2]).all())
    else:                       # outside a window
        params[int(table[0, 0]), :, 0, 3] = NAN
        params[int(table[1, 1]), :, 0, 0] = INF
        check(q, codes, params, table, lens, window=20)
    q[0, 1, 7] = INF            # a query that is not finite spoils its own row only
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    if counts is None:
        got = kv4_attention(q.to(DEVICE), codes, params, table, seq_lens, window=20)
        assert bool(torch.isfinite(got[0, [0, 2, 3]]).all()) and bool(torch.isfinite(got[1]).all())


def test_strided_queries_and_tables():
    lens = [40, 90]
    codes, params, table = make_cache(lens, 2, 64, 16, torch.float16, 34)
    fused = _vectors(2, 8, 64, torch.float16, 35).to(DEVICE)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    want = kv4_attention(fused[:, :4].contiguous(), codes, params, table, seq_lens)
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=DEVICE)
    wide[:, :table.shape[1]] = table
    assert torch.equal(kv4_attention(fused[:, :4], codes, params, wide[:, :table.shape[1]], seq_lens), want)
    turned = fused[:, :4].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(kv4_attention(turned, codes, params, table, seq_lens), want)
    odd = torch.empty((2, 4, 67), dtype=torch.float16, device=DEVICE)[:, :, 3:]
    odd.copy_(fused[:, :4])
    assert torch.equal(kv4_attention(odd, codes, params, table, seq_lens), want)


def test_no_sequences_and_no_pages():
    codes, params = allocate_kv4_cache(0, 2, 64, page_size=16, device=DEVICE)
    q = torch.ones((0, 4, 64), dtype=torch.bfloat16, device=DEVICE)
    none = torch.empty(0, dtype=torch.int32, device=DEVICE)
    assert kv4_attention(q, codes, params, none.reshape(0, 3), none).shape == (0, 4, 64)
    one = torch.ones((1, 4, 64), dtype=torch.bfloat16, device=DEVICE)
    got = kv4_attention(one, codes, params, torch.zeros((1, 3), dtype=torch.int32, device=DEVICE), torch.tensor([33], dtype=torch.int32, device=DEVICE))
    assert bool((got == 0).all())
    got = kv4_attention(one, codes, params, torch.zeros((1, 0), dtype=torch.int32, device=DEVICE), torch.tensor([33], dtype=torch.int32, device=DEVICE))
    assert bool((got == 0).all())


def test_same_bits_every_time():
    lens = [900, 33, 2100, 1, 640] * 3
    codes, params, table = make_cache(lens, 4, 128, 64, torch.bfloat16, 36)
    q = _vectors(len(lens), 16, 128, torch.bfloat16, 37).to(DEVICE)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    first = kv4_attention(q, codes, params, table, seq_lens)
    for _ in range(5):
        assert torch.equal(kv4_attention(q, codes, params, table, seq_lens), first)


def test_two_streams_and_two_captured_graphs():
    lens = [3000, 1200]
    codes, params, table = make_cache(lens, 2, 128, 64, torch.float16, 38)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    qs = [_vectors(2, 8, 128, torch.float16, 39 + i).to(DEVICE) for i in range(2)]
    want = [kv4_attention(q, codes, params, table, seq_lens) for q in qs]
    graphs, held = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(kv4_attention(q, codes, params, table, seq_lens))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    got = [None, None]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = kv4_attention(qs[i], codes, params, table, seq_lens)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    seq_lens.copy_(torch.tensor([7, 2900], dtype=torch.int32))          # lengths live on the device
    table[1, : table.shape[1] - 1] = table[0, : table.shape[1] - 1]
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, kv4_attention(q, codes, params, table, seq_lens)) for a, q in zip(held, qs))


def wide(table, page):
    """The table with room for a million keys: then a call counts as much work, and sequences with more than 32 rows go to the prompt kernel."""

    return torch.nn.functional.pad(table, (0, (1 << 20) // page), value=-1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,each,dim,page", [(2, 4, 128, 64), (1, 8, 64, 16), (2, 2, 256, 128), (1, 3, 128, 32), (4, 1, 64, 256), (1, 5, 256, 16)])
@pytest.mark.parametrize("lens,counts,window", [([300], [300], None), ([129, 700, 1000, 5], [129, 257, 300, 5], None), ([513, 1300], [512, 301], 200), ([900], [899], 1)])
def test_prompts(dtype, heads, each, dim, page, lens, counts, window):
    codes, params, table = make_cache(lens, heads, dim, page, dtype, 50)
    table = wide(table, page)
    check(_vectors(sum(counts), heads * each, dim, dtype, 51), codes, params, table, lens, counts, window=window)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,each,count", [(2, 4, 600), (2, 4, 1)])
def test_fp16_results_are_little_more_than_rounded(dim, heads, each, count):
    """Besides the rounding of the result, one of the probabilities (by their value scales): two independent errors of relative
    size r, of which the second is spread over keys with independent values, so sqrt(2) r together; 1.5 leaves 6 % for the sample.
    A third rounding, of keys or values, would make it sqrt(3) r = 1.73 r."""
    lens, counts = [1500], [count]
    codes, params, table = make_cache(lens, heads, dim, 64, torch.float16, 71)
    table = wide(table, 64)
    q = _vectors(count, heads * each, dim, torch.float16, 72)
    starts, n = torch.tensor([0, count], dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    got = kv4_attention(q.to(DEVICE), codes, params, table, n.to(DEVICE), query_starts=starts.to(DEVICE)).double()
    exact = attention(q.to(DEVICE), codes, params, table, n, starts)[0]
    rounding = (exact.half().double() - exact).norm()
    assert (got - exact).norm() < 1.5 * rounding


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("offset", [-20.0, 3.0, 1000.0])
def test_fp16_prompts_of_vectors_far_from_zero(dim, offset):
    """Minima large beside the range (and of either sign), where code * scale + minimum cancels or loses its low bits in fp16."""
    lens, counts = [333, 70], [200, 70]
    codes, params, table = make_cache(lens, 2, dim, 32, torch.float16, 73)
    table = wide(table, 32)
    params[..., 1] += offset
    check(_vectors(270, 8, dim, torch.float16, 74, 0.25), codes, params, table, lens, counts)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_of_many_sequences_beside_single_tokens(dim):
    lens, counts = [40, 700, 33, 1, 512, 90, 0, 2000] * 3, [40, 1, 9, 1, 512, 33, 3, 700] * 3
    codes, params, table = make_cache(lens, 2, dim, 32, torch.bfloat16, 52)
    table = wide(table, 32)
    check(_vectors(sum(counts), 16, dim, torch.bfloat16, 53), codes, params, table, lens, counts)


def test_prompt_with_more_queries_than_keys_and_other_scales():
    lens, counts = [100, 0, 300], [400, 300, 300]
    codes, params, table = make_cache(lens, 1, 128, 16, torch.bfloat16, 54)
    table = wide(table, 16)
    for scale in (0.5, -0.125, 0.0):
        got = check(_vectors(1000, 4, 128, torch.bfloat16, 55), codes, params, table, lens, counts, scale=scale)
        assert bool((got[:300] == 0).all()) and bool((got[400:700] == 0).all()) and bool((got[300:400] != 0).any())


def test_prompt_over_pages_that_are_not_there():
    lens, counts = [600, 400], [300, 400]
    codes, params, table = make_cache(lens, 2, 64, 16, torch.float16, 56)
    table = wide(table, 16)
    table[0, 0], table[0, 7], table[0, 36], table[1, 3:8], table[1, 24] = -1, codes.shape[0], 2 ** 31 - 1, -1, -2 ** 31
    check(_vectors(700, 8, 64, torch.float16, 57), codes, params, table, lens, counts)
    table[1] = -1
    got = check(_vectors(700, 8, 64, torch.float16, 57), codes, params, table, lens, counts)
    assert bool((got[300:] == 0).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_with_large_and_unequal_values(dim):
    lens, counts = [700], [700]
    codes, params, table = make_cache(lens, 1, dim, 64, torch.bfloat16, 58, size=4.0)
    table = wide(table, 64)
    position = torch.empty(codes.shape[0], 64, dtype=torch.long)
    for i, p in enumerate(table[0, :11].tolist()):
        position[p] = torch.arange(64) + 64 * i
    scale = torch.where(position % 7 == 0, 1e-4, torch.where(position % 7 == 3, 1e4, 1.0)) * torch.where(position < 300, 1e-6, 1.0)
    params[:, 1] *= scale.to(DEVICE)[:, None, :, None].to(params.dtype)
    params[:, 0] *= torch.where(position < 200, 1e5, 1.0).to(DEVICE)[:, None, :, None].to(params.dtype)
    q = _vectors(700, 4, dim, torch.bfloat16, 59)
    q[100:200] *= 1e-8
    q[300:400] *= 30
    q[401] = 0
    check(q, codes, params, table, lens, counts)


def test_prompt_rows_do_not_meet_what_they_do_not_see():
    """NaN and infinities in later keys and values of the same tile, in unused rows of pages, and in single queries."""

    lens, counts = [500], [400]
    codes, params, table = make_cache(lens, 2, 128, 64, torch.bfloat16, 60)
    table = wide(table, 64)
    q = _vectors(400, 8, 128, torch.bfloat16, 61).to(DEVICE)
    q[7, 3, 5] = INF
    clean = params.clone()
    for at, which, head, value in ((450, 0, 0, NAN), (460, 1, 0, NAN), (470, 1, 1, INF), (300, 0, 1, INF)):
        params[int(table[0, at // 64]), which, head, at % 64] = value
    seq_lens, starts = (torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in (lens, [0, 400]))
    got, want = (kv4_attention(q, codes, x, table, seq_lens, query_starts=starts) for x in (params, clean))
    sees = torch.zeros((400, 2), dtype=torch.bool, device=DEVICE)
    sees[350:, 0] = True         # query i stands at key 100 + i
    sees[200:, 1] = True
    sees = sees.repeat_interleave(4, 1)
    sees[7, 3] = True
    assert bool(torch.isfinite(want[~sees]).all()) and bool(torch.isnan(got[sees]).all())
    assert torch.equal(got[~sees], want[~sees])


def test_prompt_in_place_of_rows_and_graph():
    """Rows of no sequence stay, strided queries give the bits of contiguous ones, and a captured call follows the lengths on the device."""

    lens, counts = [400, 350], [300, 260]
    codes, params, table = make_cache(lens, 2, 128, 32, torch.float16, 62)
    table = wide(table, 32)
    fused = _vectors(600, 12, 128, torch.float16, 63).to(DEVICE)
    q = fused[:, :8]
    seq_lens, starts = torch.tensor(lens, dtype=torch.int32, device=DEVICE), torch.tensor([10, 310, 570], dtype=torch.int32, device=DEVICE)
    out = torch.full((600, 8, 128), 7.0, dtype=torch.float16, device=DEVICE)
    kv4_attention(q, codes, params, table, seq_lens, query_starts=starts, out=out)
    assert bool((out[:10] == 7).all()) and bool((out[570:] == 7).all()) and not bool((out[10:570] == 7).all(-1).any())
    again = kv4_attention(q.contiguous(), codes, params, table, seq_lens, query_starts=starts)
    assert torch.equal(again[10:570], out[10:570])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = kv4_attention(q, codes, params, table, seq_lens, query_starts=starts)
    seq_lens.copy_(torch.tensor([310, 340], dtype=torch.int32))
    starts.copy_(torch.tensor([0, 5, 345], dtype=torch.int32))
    graph.replay()
    want = kv4_attention(q, codes, params, table, seq_lens, query_starts=starts)
    assert torch.equal(held[:345], want[:345]) and native.workspace_status(DEVICE) == 0


@pytest.mark.parametrize("lens,counts", [([3000], [70]), ([700, 2000, 64], [65, 300, 9]), ([100] * 40, [60] * 40)])
def test_prompt_kernel_beside_the_other_one(lens, counts):
    """The same call by either kernel (the width of the table chooses): both within their bounds; items that several CTAs share among them."""

    codes, params, table = make_cache(lens, 2, 128, 64, torch.bfloat16, 64)
    q = _vectors(sum(counts), 8, 128, torch.bfloat16, 65)
    for t in (table, wide(table, 64)):
        check(q, codes, params, t, lens, counts)


def test_same_prompt_bits_every_time():
    lens, counts = [1500, 900, 300], [700, 900, 20]
    codes, params, table = make_cache(lens, 2, 128, 64, torch.bfloat16, 66)
    q = _vectors(sum(counts), 8, 128, torch.bfloat16, 67).to(DEVICE)
    seq_lens, starts = torch.tensor(lens, dtype=torch.int32, device=DEVICE), torch.tensor([0, 700, 1600, 1620], dtype=torch.int32, device=DEVICE)
    first = kv4_attention(q, codes, params, wide(table, 64), seq_lens, query_starts=starts)
    for _ in range(10):
        assert torch.equal(kv4_attention(q, codes, params, wide(table, 64), seq_lens, query_starts=starts), first)


def test_native_path_and_python_path_give_the_same():
    from xqt_b200.ops import kv4, rotary

    lens = [300, 77]
    codes, params, table = make_cache(lens, 2, 128, 32, torch.bfloat16, 68)
    x = _vectors(2, 12, 128, torch.bfloat16, 69).to(DEVICE)
    seq_lens, slots, positions = torch.tensor(lens, dtype=torch.int32, device=DEVICE), torch.tensor([5, 40], device=DEVICE), torch.tensor([299, 76], device=DEVICE)
    frequencies, weight = rotary.rotary_frequencies(128, device=DEVICE)[0], torch.rand(128, generator=seeded(70)).to(DEVICE)

    def run():
        q, k = rotary.qk_norm_rope(x[:, :8], x[:, 8:10], positions, frequencies, q_weight=weight, k_weight=weight, interleaved=True)
        cache = [t.clone() for t in (codes, params)]
        kv4_append(k, x[:, 10:], *cache, slots)
        return (q, k, *cache, *kv4_gather(*cache, slots), kv4_attention(q, *cache, table, seq_lens, window=50, scale=0.1))

    run()
    assert kv4._native is not None and rotary._native is not None
    fast = run()
    kv4._native = rotary._native = None
    for a, b in zip(fast, run()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


_FIRST_CALL_IN_A_CAPTURE = """
import os, sys
sys.path.insert(0, os.environ["XQT_ROOT"]); sys.path.insert(0, os.path.join(os.environ["XQT_ROOT"], "tests"))
import torch
from test_kv4_gpu import DEVICE, _vectors, make_cache, wide
from xqt_b200 import native
from xqt_b200.ops.kv4 import kv4_attention
codes, params, table = make_cache([200, 90], 2, 128, 32, torch.bfloat16, 1)
q = _vectors(160, 8, 128, torch.bfloat16, 2).to(DEVICE)
lens, starts = (torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in ([200, 90], [0, 100, 160]))
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    held = kv4_attention(q, codes, params, wide(table, 32), lens, query_starts=starts), kv4_attention(q[:2], codes, params, table, lens)
graph.replay()
want = kv4_attention(q, codes, params, wide(table, 32), lens, query_starts=starts), kv4_attention(q[:2], codes, params, table, lens)
assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]) and native.workspace_status(DEVICE) == 0
print("the same")
"""


def test_first_call_of_a_process_in_a_capture():
    import os
    import subprocess
    import sys

    from conftest import ROOT

    done = subprocess.run([sys.executable, "-c", _FIRST_CALL_IN_A_CAPTURE], env={**os.environ, "XQT_ROOT": str(ROOT)}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]


def test_many_short_sequences():
    lens = [(7 * i) % 50 for i in range(700)]
    codes, params, table = make_cache(lens, 1, 64, 16, torch.float16, 41)
    check(_vectors(len(lens), 2, 64, torch.float16, 42), codes, params, table, lens)


def test_out_is_checked():
    codes, params = allocate_kv4_cache(1, 2, 64, page_size=16, device=DEVICE)
    q = torch.ones((1, 4, 64), dtype=torch.bfloat16, device=DEVICE)
    table, seq_lens = torch.zeros((1, 1), dtype=torch.int32, device=DEVICE), torch.ones(1, dtype=torch.int32, device=DEVICE)
    for bad in (q.half(), torch.ones((2, 4, 64), dtype=torch.bfloat16, device=DEVICE), torch.ones((1, 4, 128), dtype=torch.bfloat16, device=DEVICE)[..., ::2]):
        with pytest.raises(XQTBackendError, match="out"):
            kv4_attention(q, codes, params, table, seq_lens, out=bad)
