"""Norm and rotation of query and key heads against the formula in 64 bits."""

from __future__ import annotations

import pytest
import torch

from attention_reference import norm_rope, rope_bound
from conftest import seeded
from xqt_b200.errors import XQTBackendError
from xqt_b200.ops.rotary import qk_norm_rope, rotary_frequencies

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)


def _draw(tokens, heads, dim, dtype, seed):
    return (torch.randn((tokens, heads, dim), generator=seeded(seed)) * 1.5).to(dtype).to(DEVICE)


def _close(got, x, *args, **kwargs):
    want, size = norm_rope(x, *args, **kwargs)
    error = (got.cpu().double() - want).abs()
    assert bool((error <= rope_bound(want, size, got.dtype)).all()), float((error - rope_bound(want, size, got.dtype)).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,q_heads,k_heads,dim,rotary", [
    (1, 32, 8, 128, 128), (3, 5, 1, 64, 64), (17, 4, 4, 96, 96), (9, 3, 1, 80, 48), (5, 7, 1, 256, 256), (130, 2, 1, 128, 64), (2, 1, 1, 16, 16),
    (4, 3, 2, 208, 112), (33, 40, 8, 128, 128)])
def test_norm_and_rotation(dtype, interleaved, tokens, q_heads, k_heads, dim, rotary):
    q, k = _draw(tokens, q_heads, dim, dtype, 1), _draw(tokens, k_heads, dim, dtype, 2)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=seeded(3))
    frequencies, axes = rotary_frequencies(rotary, theta=1e6)
    assert axes is None
    qw, kw = (1 + 0.3 * torch.randn((2, dim), generator=seeded(4))).to(dtype)
    got = qk_norm_rope(q, k, positions.to(DEVICE), frequencies.to(DEVICE), q_weight=qw.to(DEVICE), k_weight=kw.to(DEVICE), interleaved=interleaved, eps=1e-5)
    _close(got[0], q, positions, frequencies, weight=qw, eps=1e-5, interleaved=interleaved)
    _close(got[1], k, positions, frequencies, weight=kw, eps=1e-5, interleaved=interleaved)


@pytest.mark.parametrize("form", ["sections", "ladders", "odd"])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_several_axes_without_norm(form, wide):
    q, k = _draw(57, 6, 128, torch.bfloat16, 5), _draw(57, 2, 128, torch.bfloat16, 6)
    positions = torch.randint(-3000, 3000, (3, 57), generator=seeded(7)).to(wide)
    if form == "sections":
        frequencies, axes = rotary_frequencies(128, sections=(16, 24, 24))
    elif form == "ladders":
        frequencies, axes = rotary_frequencies(128, ladders=(16, 56, 56))
    else:       # axes in turn, some of them outside
        frequencies, axes = rotary_frequencies(128)
        axes = torch.arange(-1, 63, dtype=torch.int32) % 5
    interleaved = form != "sections"
    got = qk_norm_rope(q, k, positions.to(DEVICE), frequencies.to(DEVICE), axes=axes.to(DEVICE), interleaved=interleaved)
    _close(got[0], q, positions, frequencies, axes=axes, interleaved=interleaved)
    _close(got[1], k, positions, frequencies, axes=axes, interleaved=interleaved)


@pytest.mark.parametrize("which", ["q", "k"])
def test_one_side_normed(which):
    q, k = _draw(11, 4, 128, torch.float16, 8), _draw(11, 4, 128, torch.float16, 9)
    frequencies, _ = rotary_frequencies(128)
    weight = torch.rand((128,), generator=seeded(10)) + 0.5
    positions = torch.arange(11)
    got = qk_norm_rope(q, k, positions.to(DEVICE), frequencies.to(DEVICE), **{f"{which}_weight": weight.to(DEVICE)})
    _close(got[0], q, positions, frequencies, weight=weight if which == "q" else None)
    _close(got[1], k, positions, frequencies, weight=weight if which == "k" else None)


@pytest.mark.parametrize("position", [0, 1, 2 ** 24 + 1, 2 ** 31 - 1, -1, -2 ** 31, 2 ** 40 + 7])
def test_far_positions(position):
    q = _draw(1, 2, 64, torch.float16, 11)
    frequencies, _ = rotary_frequencies(64)
    # frequencies of a turn that doubles hold exactly up to 2^40 positions: multiples of 2^-10 turns would not test the wrap, so
    # the reference takes the turns as the kernel does, frequency / (2 pi) in 64 bits, and whole-number arithmetic from there
    from fractions import Fraction
    import math
    fraction = [Fraction(float(f) * 0.15915494309189535) for f in frequencies]
    angle = torch.tensor([float((f * position) % 1) * 2 * math.pi for f in fraction], dtype=torch.float64)
    x = q.cpu().double()
    a, b = x[..., :32], x[..., 32:]
    want = torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    got, none = qk_norm_rope(q, None, torch.tensor([position], device=DEVICE), frequencies.to(DEVICE))
    assert none is None
    # the fraction of a turn is held to 2^-53 (of a double below 1): 2 pi 2^-53 |position| more
    bound = rope_bound(want, size, torch.float16) + size * 7 * 2.0 ** -53 * abs(position)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_strided_inputs_outputs_and_in_place():
    fused = _draw(21, 4 + 2 + 2, 128, torch.bfloat16, 12)
    q, k = fused[:, :4], fused[:, 4:6]
    frequencies, _ = rotary_frequencies(128)
    positions = torch.arange(21, device=DEVICE)
    weight = torch.ones(128, device=DEVICE, dtype=torch.bfloat16)
    args = dict(q_weight=weight, k_weight=weight)
    want = qk_norm_rope(q.contiguous(), k.contiguous(), positions, frequencies.to(DEVICE), **args)
    got = qk_norm_rope(q, k, positions, frequencies.to(DEVICE), **args)
    # heads before tokens, channels off 16 bytes, positions with a stride
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty((21, 2, 131), dtype=torch.bfloat16, device=DEVICE)[:, :, 3:]
    odd.copy_(k)
    again = qk_norm_rope(turned, odd, torch.stack((positions, positions), 1).reshape(-1)[::2], frequencies.to(DEVICE), **args)
    rest = fused[:, 6:].clone()
    qk_norm_rope(q, k, positions, frequencies.to(DEVICE), out=(q, k), **args)
    for a, b, c, w in zip(got, again, (q, k), want):
        assert torch.equal(a, w) and torch.equal(b, w) and torch.equal(c, w)
    assert torch.equal(fused[:, 6:], rest)


def test_zeros_infinities_and_nan_stay_in_their_head():
    q = _draw(3, 3, 128, torch.float16, 13)
    clean = q.clone()
    q[0, 1, 5], q[1, 0, 100], q[2, 2] = float("inf"), float("nan"), 0
    frequencies, _ = rotary_frequencies(128)
    weight = torch.ones(128, device=DEVICE)
    run = lambda x: qk_norm_rope(x, None, torch.arange(3, device=DEVICE), frequencies.to(DEVICE), q_weight=weight)[0]  # noqa: E731
    got, want = run(q), run(clean)
    touched = torch.zeros((3, 3), dtype=torch.bool)
    touched[0, 1] = touched[1, 0] = touched[2, 2] = True
    assert torch.equal(got[~touched.to(DEVICE)], want[~touched.to(DEVICE)])
    assert bool((got[2, 2] == 0).all()) and not bool(torch.isfinite(got[0, 1]).all()) and bool(torch.isnan(got[1, 0]).all())


def test_nothing_to_do_and_no_rotation():
    frequencies = torch.empty(0, dtype=torch.float64, device=DEVICE)
    q = _draw(4, 2, 48, torch.bfloat16, 14)
    got, _ = qk_norm_rope(q, None, torch.arange(4, device=DEVICE), frequencies)
    assert torch.equal(got, q)
    got = qk_norm_rope(q[:0], q[:0], torch.arange(0, device=DEVICE), frequencies)
    assert got[0].shape == got[1].shape == (0, 2, 48)


def test_many_tokens_equal_few():
    """Tokens past one block, and the head counts per group that their number chooses, give the bits of single calls."""

    q, k = _draw(3001, 8, 128, torch.bfloat16, 15), _draw(3001, 2, 128, torch.bfloat16, 16)
    frequencies, _ = rotary_frequencies(128)
    weight = torch.rand((128,), generator=seeded(17)).to(DEVICE)
    positions = torch.arange(3001, device=DEVICE) * 7
    got = qk_norm_rope(q, k, positions, frequencies.to(DEVICE), q_weight=weight, k_weight=weight)
    for at in (0, 1, 1499, 3000):
        one = qk_norm_rope(q[at:at + 1], k[at:at + 1], positions[at:at + 1], frequencies.to(DEVICE), q_weight=weight, k_weight=weight)
        assert torch.equal(got[0][at:at + 1], one[0]) and torch.equal(got[1][at:at + 1], one[1])


def test_other_stream_and_captured_graph():
    q = _draw(6, 4, 128, torch.float16, 18)
    frequencies = rotary_frequencies(128)[0].to(DEVICE)
    positions = torch.arange(6, device=DEVICE)
    want = qk_norm_rope(q, q, positions, frequencies)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = qk_norm_rope(q, q, positions, frequencies)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = qk_norm_rope(q, q, positions, frequencies)
    positions += 5
    graph.replay()
    want = qk_norm_rope(q, q, positions, frequencies)
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


def test_refusals_on_the_gpu():
    q = _draw(2, 2, 128, torch.float16, 19)
    frequencies, positions = rotary_frequencies(128)[0].to(DEVICE), torch.arange(2, device=DEVICE)
    with pytest.raises(XQTBackendError, match="output"):
        qk_norm_rope(q, None, positions, frequencies, out=(q[:1].expand(2, 2, 128), None))
    with pytest.raises(XQTBackendError, match="outputs go with inputs"):
        qk_norm_rope(q, None, positions, frequencies, out=(q, q))
    with pytest.raises(XQTBackendError, match="device"):
        qk_norm_rope(q, None, positions.cpu(), frequencies)
