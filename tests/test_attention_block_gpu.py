"""The operators between the projections as a decoder layer uses them: a prompt, single tokens, drafted tokens, through one 4-bit cache."""

from __future__ import annotations

import pytest
import torch

from attention_reference import attention, norm_rope
from conftest import seeded
from oracle import w4a16 as oracle
from xqt_b200 import quantize
from xqt_b200.errors import XQTBackendError
from xqt_b200.kernel_spec import get_kernel
from xqt_b200.ops.attention import W4A16Attention
from xqt_b200.ops.kv4 import kv4_append, kv4_attention, kv4_gather
from xqt_b200.ops.rotary import qk_norm_rope, rotary_frequencies

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
HIDDEN, HEADS, KV, DIM, PAGE = 1024, 8, 2, 128, 32


def _block(dtype, seed=1, **options):
    gen = seeded(seed)
    weights = [quantize.quantize_w4_asymmetric(torch.randn((n, k), generator=gen) * k ** -0.5, group_size=128)
               for n, k in ((HEADS * DIM, HIDDEN), (KV * DIM, HIDDEN), (KV * DIM, HIDDEN), (HIDDEN, HEADS * DIM))]
    norms = 1 + 0.2 * torch.randn((2, DIM), generator=gen)
    frequencies, _ = rotary_frequencies(DIM, theta=1e6)
    block = W4A16Attention(*weights, kv_heads=KV, head_dim=DIM, frequencies=frequencies, q_norm=norms[0], k_norm=norms[1], device=DEVICE, dtype=dtype, **options)
    dense = [oracle.dequantize(w.qweight, w.scales, w.zero_points, k=w.metadata.logical_shape[1], padded_k=w.metadata.logical_shape[1], group_size=128,
                              signed=False).double() for w in weights]
    return block, dense, norms, frequencies


def _steps():
    """(tokens of each of two sequences, their lengths behind the step): a prompt and a shorter one, tokens, drafts, one sequence alone."""

    return [([75, 40], [75, 40]), ([1, 1], [76, 41]), ([1, 1], [77, 42]), ([4, 3], [81, 45]), ([0, 1], [81, 46]), ([1, 0], [82, 46])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [None, 30])
def test_a_run_of_steps(dtype, window):
    block, dense, norms, frequencies = _block(dtype, window=window)
    cache = block.allocate_cache(12, PAGE)
    table = torch.tensor([[3, 9, 1, -1], [7, 0, -1, -1]], dtype=torch.int32, device=DEVICE)
    gen = seeded(2)
    for counts, lens in _steps():
        tokens = sum(counts)
        x = torch.randn((tokens, HIDDEN), generator=gen).to(dtype).to(DEVICE)
        positions = torch.cat([torch.arange(n - m, n) for m, n in zip(counts, lens)])
        owner = torch.cat([torch.full((m,), b) for b, m in enumerate(counts)]).long()
        slots = (table.cpu().long()[owner, positions // PAGE] * PAGE + positions % PAGE).to(DEVICE)
        seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
        starts = None if counts == [1, 1] else torch.tensor([0, counts[0], tokens], dtype=torch.int32, device=DEVICE)
        before = [t.clone() for t in cache]
        got = block(x, positions.to(DEVICE), cache, slots, table, seq_lens, starts)

        # the same operators called one by one give the same bits
        heads = block.qkv(x).view(tokens, HEADS + 2 * KV, DIM)
        q, k = qk_norm_rope(heads[:, :HEADS], heads[:, HEADS:HEADS + KV], positions.to(DEVICE), block.frequencies, q_weight=block.q_norm, k_weight=block.k_norm)
        kv4_append(k, heads[:, HEADS + KV:], *before, slots)
        assert torch.equal(before[0], cache[0]) and torch.equal(before[1], cache[1])
        mid = kv4_attention(q, *cache, table, seq_lens, query_starts=starts, window=window)
        assert torch.equal(block.o(mid.view(tokens, HEADS * DIM)), got)

        # what the cache holds is what the projections give, to half a code step (scale / 2, and the clamp's 15 half steps of the type) and the
        # rounding of three operators in the type
        eps = torch.finfo(dtype).eps
        xd = x.cpu().double()
        kd, _ = norm_rope((xd @ dense[1].T).view(tokens, KV, DIM), positions, frequencies, weight=norms[1])
        vd = (xd @ dense[2].T).view(tokens, KV, DIM)
        for held, want in zip(kv4_gather(*cache, slots), (kd, vd)):
            step = (want.amax(-1, keepdim=True) - want.amin(-1, keepdim=True)) / 15
            assert bool(((held.cpu().double() - want).abs() <= step * (0.5 + 15 * eps) + 4 * eps * want.abs().amax(-1, keepdim=True)).all())

        # and the block's result is that of 64-bit operators over the cache as it is.  Rounding in between: the query projection, the rotated
        # query, the attention output and the result, each to eps / 2 of its size; queries' errors reach the scores, whose size is below 8 here
        qd, _ = norm_rope((xd @ dense[0].T).view(tokens, HEADS, DIM), positions, frequencies, weight=norms[0])
        middle, _ = attention(qd, cache[0].cpu(), cache[1].cpu(), table.cpu(), torch.tensor(lens), None if starts is None else starts.cpu(), window=window)
        want = middle.reshape(tokens, HEADS * DIM) @ dense[3].T
        assert oracle.rel_l2(got.cpu(), want) <= 8 * eps


def test_no_tokens_and_refusals():
    block, _, _, frequencies = _block(torch.bfloat16)
    cache = block.allocate_cache(2)
    none = torch.empty(0, dtype=torch.int64, device=DEVICE)
    got = block(torch.empty((0, HIDDEN), dtype=torch.bfloat16, device=DEVICE), none, cache, none, torch.zeros((0, 1), dtype=torch.int32, device=DEVICE),
                torch.empty(0, dtype=torch.int32, device=DEVICE))
    assert got.shape == (0, HIDDEN)
    with pytest.raises(XQTBackendError, match="tokens, hidden"):
        block(torch.empty((1, HIDDEN), dtype=torch.float16, device=DEVICE), none, cache, none, none, none)
    w = lambda n, k: quantize.quantize_w4_asymmetric(torch.zeros((n, k)), group_size=128)  # noqa: E731
    for q, k, v, o, heads, dim in ((768, 256, 256, 768, 2, 128), (512, 256, 256, 512, 2, 96), (512, 128, 256, 512, 2, 128), (512, 256, 256, 256, 2, 128)):
        if (q, heads, dim) == (768, 2, 128):
            heads = 4                       # 6 query heads on 4
        with pytest.raises(XQTBackendError):
            W4A16Attention(w(q, 256), w(k, 256), w(v, 256), w(256, o), kv_heads=heads, head_dim=dim, frequencies=frequencies, device=DEVICE)


def test_decode_step_in_a_graph():
    """One captured step serves later steps: positions, slots and lengths are read from the device."""

    block, _, _, _ = _block(torch.bfloat16)
    cache = block.allocate_cache(6, PAGE)
    eager = [t.clone() for t in cache]
    table = torch.tensor([[5, 0], [2, 4]], dtype=torch.int32, device=DEVICE)
    x = torch.zeros((2, HIDDEN), dtype=torch.bfloat16, device=DEVICE)
    positions, slots = torch.zeros(2, dtype=torch.int64, device=DEVICE), torch.zeros(2, dtype=torch.int64, device=DEVICE)
    seq_lens = torch.ones(2, dtype=torch.int32, device=DEVICE)
    run = lambda c: block(x, positions, c, slots, table, seq_lens)  # noqa: E731
    slots.copy_(table[:, 0].long() * PAGE)
    run(eager)
    for t in eager:
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(cache)
    for step in range(40):
        x.copy_(torch.randn((2, HIDDEN), generator=seeded(100 + step)).to(torch.bfloat16))
        positions.fill_(step)
        slots.copy_(table[:, step // PAGE].long() * PAGE + step % PAGE)
        seq_lens.fill_(step + 1)
        graph.replay()
        assert torch.equal(held, run(eager))
    assert torch.equal(cache[0], eager[0]) and torch.equal(cache[1], eager[1])


def test_kernel_namespace():
    assert get_kernel("attention.qk_norm_rope") is qk_norm_rope and get_kernel("attention.kv4_attention") is kv4_attention
    assert get_kernel("attention.kv4_append") is kv4_append and get_kernel("attention.kv4_gather") is kv4_gather
