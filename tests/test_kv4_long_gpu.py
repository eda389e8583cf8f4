"""Attention over the 4-bit cache in long contexts: what a sum of many small terms has to keep."""

from __future__ import annotations

import math

import pytest
import torch

from attention_reference import attention
from conftest import seeded
from xqt_b200 import native
from xqt_b200.ops.kv4 import kv4_attention

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
PAGE = 64


def long_prompt(keys, dim, dtype, queries, exponent=None, seed=81, heads=None):
    """A key head per SM, so that every one has whole items (unless ``heads`` says otherwise); the tables go round 64 pages.  Values lie in [0.53, 1.47] with a mean of 1.  With ``exponent`` the first key is
    2 ** exponent times as probable as the others are on average, and its values are 0.  -> arguments, and those of the first two heads for the reference."""

    heads = heads or torch.cuda.get_device_properties(0).multi_processor_count
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    codes = torch.randint(0, 256, (65, 2, heads, PAGE, dim // 2), dtype=torch.uint8, device=DEVICE, generator=gen)
    params = torch.empty((65, 2, heads, PAGE, 2), dtype=dtype, device=DEVICE)
    for which, step, mean in ((0, 1 / 16, 0.0), (1, 1 / 16, 1.0)):
        params[:, which, ..., 0], params[:, which, ..., 1] = step, mean - 7.5 * step
    q = torch.randn((queries, heads, dim), generator=seeded(seed + 1)) / math.sqrt(dim)
    table = (torch.arange(keys // PAGE, dtype=torch.int32) % 64).reshape(1, -1)
    if exponent is not None:
        params[64, :, :, 0, 0], params[64, :, :, 0, 1] = 1.0, 0.0
        codes[64, 0, :, 0], codes[64, 1, :, 0] = 0x01, 0          # 1 in the even channels
        table[0, 0] = 64
        q[..., 0::2] += 2 * exponent * math.log(2) / dim
        q[..., 1::2] -= 2 * exponent * math.log(2) / dim          # no score for what the other keys have on average
    q = q.to(dtype).to(DEVICE)
    lens, starts = torch.tensor([keys], dtype=torch.int32), torch.tensor([0, queries], dtype=torch.int32)
    wide = torch.nn.functional.pad(table, (0, (1 << 20) // PAGE), value=-1)      # so wide that the prompt kernel is taken
    return (q, codes, params, wide.to(DEVICE), lens.to(DEVICE), starts.to(DEVICE)), (q[:, :2], codes[:, :, :2], params[:, :, :2], table, lens, starts)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("exponent", [16, 21, 26])
def test_many_weak_keys_beside_a_strong_one(dim, exponent):
    """Probabilities 2^-16 to 2^-26 of the row's largest, whose key has values of 0: the result is what the weak ones leave."""
    keys, queries = 16384, 40
    call, small = long_prompt(keys, dim, torch.float16, queries, exponent)
    got = kv4_attention(*call[:5], query_starts=call[5], scale=1.0)[:, :2].double()
    want, bound = attention(*small, scale=1.0)
    # Besides the bound for one rounding of the probabilities relative to them: against 2^7 for the row's largest a half is held to 2^-25, so each
    # probability to 2^-32 of it; independent errors, weighted by values of at most 1.5 (7 deviations: see the reference).  And sums that the tensor core
    # cuts off: at most 2^-23 each of the running sum, 8 of them in a chunk of 64 keys.
    subnormal = 7 * 2.0 ** -32 * math.sqrt(keys) * 1.5
    bound = bound + subnormal + keys / 64 * 8 * 2.0 ** -23 * want.abs()
    assert float((bound / want.abs()).max()) < 1 / 8             # some rows' strong key is 2^29 times as probable: their bound still says something
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1, f"{worst} bounds; {float(((got - want).abs() / want.abs()).max())} of the result"
    assert native.workspace_status(DEVICE) == 0


def summed(dtype, want):
    """What the tensor core's sums may lose: of each product the bits below 2^-24 of the running sum, which is of one sign here, in runs of 4096 keys with
    two products each (fp16) or of 16,384 with one (bf16)."""
    return (2 * 4096 if dtype == torch.float16 else 16384) * 2.0 ** -24 * want.abs()


@pytest.mark.parametrize("dtype,dim,keys", [(torch.float16, 64, 131072), (torch.float16, 128, 131072), (torch.float16, 256, 131072), (torch.bfloat16, 64, 1 << 20)])
def test_long_sums_of_values_of_one_sign(dtype, dim, keys):
    call, small = long_prompt(keys, dim, dtype, 40)
    got = kv4_attention(*call[:5], query_starts=call[5], scale=0.25)[:, :2].double()
    want, bound = attention(*small, scale=0.25, rounded=torch.float16)
    worst = float(((got - want).abs() / (bound + summed(dtype, want))).max())
    assert worst <= 1, f"{worst} bounds"
    assert native.workspace_status(DEVICE) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("keys", [4096, 16384, 20032])
@pytest.mark.parametrize("heads,window", [(None, None), (100, None), (100, 9000)])
def test_runs_of_keys_in_whole_and_in_shared_items(dtype, dim, keys, heads, window):
    """Around the lengths at which a sum is put aside, with items of one CTA and of two; hidden pages so that whole runs see nothing, and queries that are not finite."""
    call, small = long_prompt(keys, dim, dtype, 70, heads=heads)
    call[0][5, 1, 3] = float("inf")
    for hidden in (None, slice(0, 70), slice(max(keys // PAGE - 70, 0), keys // PAGE)):
        table, short = call[3].clone(), small[3].clone()
        if hidden is not None:
            table[:, hidden] = -1
            short[:, hidden] = -1
        got = kv4_attention(*call[:3], table, call[4], query_starts=call[5], window=window)[:, :2].double()
        want, bound = attention(*small[:3], short, *small[4:], rounded=torch.float16, window=window)
        sees = torch.arange(keys).reshape(-1, PAGE)[(short[0] >= 0)]
        last = torch.arange(keys - 70, keys)
        nothing = torch.tensor([not bool(((sees <= i) & (sees > i - (window or keys))).any()) for i in last.tolist()])
        assert bool((got[nothing.to(DEVICE)] == 0).all())
        spoilt = torch.zeros((70, 2), dtype=torch.bool, device=DEVICE)
        spoilt[5, 1] = not bool(nothing[5])
        assert bool(torch.isnan(got[spoilt]).all()) and bool(torch.isfinite(got[~spoilt]).all())
        over = (got - want).abs()[~spoilt] - (bound + summed(dtype, want))[~spoilt]
        assert bool((over <= 0).all()), f"{float(over.max())} over"
    first = kv4_attention(*call[:5], query_starts=call[5], window=window)
    for _ in range(3):
        again = kv4_attention(*call[:5], query_starts=call[5], window=window)
        assert torch.equal(again.view(torch.uint8), first.view(torch.uint8))
    assert native.workspace_status(DEVICE) == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts,dtype,ratio", [([600, 300], torch.bfloat16, 24), ([600, 300], torch.float16, 12), ([7, 5], torch.bfloat16, 12), ([7, 5], torch.float16, 12)])
def test_large_finite_vectors_that_a_row_does_not_see(dim, counts, dtype, ratio):
    """Later keys and values 2^ratio times as large as their neighbours, in the same chunks: rows before them are as exact as without."""
    from test_kv4_gpu import _vectors, make_cache, wide

    lens = [600, 900]
    codes, params, table = make_cache(lens, 2, dim, 64, dtype, 83)
    large = {0: [595, 598, 599], 1: [897, 899]}
    for b, keys in large.items():
        for key in keys:
            params[int(table[b, key // 64]), :, :, key % 64] *= 2.0 ** ratio
    assert bool(torch.isfinite(params[int(table[0, 9]), :, :, :24]).all())
    q = _vectors(sum(counts), 8, dim, dtype, 84).to(DEVICE)
    seq_lens, starts = torch.tensor(lens, dtype=torch.int32), torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32)
    got = kv4_attention(q, codes, params, wide(table, 64), seq_lens.to(DEVICE), query_starts=starts.to(DEVICE)).double()
    want, bound = attention(q, codes, params, table, seq_lens, starts, rounded=torch.float16 if max(counts) > 32 else None)
    clear = torch.tensor([lens[b] - counts[b] + i < large[b][0] for b in (0, 1) for i in range(counts[b])], device=DEVICE)
    # the bound takes a sequence's largest key for all of its rows: the rows before it get theirs from a cache without the large ones
    plain = params.clone()
    for b, keys in large.items():
        for key in keys:
            plain[int(table[b, key // 64]), :, :, key % 64] *= 2.0 ** -ratio
    same, bound = attention(q, codes, plain, table, seq_lens, starts, rounded=torch.float16 if max(counts) > 32 else None)
    assert bool(clear.any()) and not bool(clear.all()) and torch.equal(want[clear], same[clear])
    over = (got - same).abs()[clear] - bound[clear]
    assert bool((over <= 0).all()), f"{float(over.max())} over a bound of {float(bound[clear].max())}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_million_keys_beside_a_strong_one_for_single_tokens(dtype):
    """Single tokens: 2^20 keys at 2^-24 of one whose values are half of theirs, in items of one CTA: sums to which each weak key adds half of their last bit."""
    keys, dim, each = 1 << 20, 64, 4
    heads = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    gen = torch.Generator(device=DEVICE).manual_seed(85)
    codes = torch.randint(0, 256, (65, 2, heads, PAGE, dim // 2), dtype=torch.uint8, device=DEVICE, generator=gen)
    params = torch.empty((65, 2, heads, PAGE, 2), dtype=dtype, device=DEVICE)
    params[:, 0, ..., 0], params[:, 0, ..., 1] = 2.0 ** -6, -7.5 * 2.0 ** -6
    params[:, 1, ..., 0], params[:, 1, ..., 1] = 1 / 16, 2 - 7.5 / 16
    codes[64, 0, :, 0], params[64, 0, :, 0, 0], params[64, 0, :, 0, 1] = 0x0F, 1 / 15, 0.0       # 1 in the even channels
    codes[64, 1, :, 0], params[64, 1, :, 0, 0], params[64, 1, :, 0, 1] = 0, 1.0, 1.0
    q = torch.zeros((1, heads * each, dim))
    q[..., 0::2] = 24 * math.log(2) / (dim // 2)
    q = q.to(dtype).to(DEVICE)
    table = (torch.arange(keys // PAGE, dtype=torch.int32) % 64).reshape(1, -1)
    table[0, 0] = 64
    lens = torch.tensor([keys], dtype=torch.int32)
    got = kv4_attention(q, codes, params, table.to(DEVICE), lens.to(DEVICE), scale=1.0)[:, :2 * each].double()
    want, bound = attention(q[:, :2 * each], codes[:, :, :2], params[:, :, :2], table, lens, scale=1.0)
    assert bool((bound < 2 * torch.finfo(dtype).eps / 2 * want.abs()).all())
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1, f"{worst} bounds"
