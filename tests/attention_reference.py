"""Plain 64-bit forms of the operators between the QKV and output projections, and the error bounds their kernels are held to."""

from __future__ import annotations

import math

import torch


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def norm_rope(x, positions, frequencies, axes=None, weight=None, eps=1e-6, interleaved=False):
    """-> (result, bound on |result before its last rounding| errors of the fp32 arithmetic) in fp64 on the CPU."""

    x = x.detach().cpu().double()
    positions = positions.cpu().reshape(-1, positions.shape[-1])
    pairs = frequencies.shape[0]
    owner = [0] * pairs if axes is None else [min(max(int(a), 0), positions.shape[0] - 1) for a in axes.cpu()]
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.cpu().double()
    size = x.abs().clone()
    y = x.clone()
    for j in range(pairs):
        lo, hi = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
        turn = float(frequencies[j]) / (2 * math.pi)
        angle = torch.tensor([math.fmod(int(p) * turn, 1.0) * 2 * math.pi for p in positions[owner[j]]], dtype=torch.float64)[:, None]
        a, b = x[..., lo], x[..., hi]
        y[..., lo] = a * angle.cos() - b * angle.sin()
        y[..., hi] = a * angle.sin() + b * angle.cos()
        size[..., lo] = size[..., hi] = a.abs() + b.abs()
    return y, size


def rope_bound(y, size, dtype):
    # one rounding to dtype (half a step; 2^-25 is half the spacing of fp16 subnormals), and fp32: norm (the sum of up to 256
    # squares, rsqrt, two products), sine and cosine to 2^-23, two products and a sum -- below 2^-19 of the pair's size
    return half_step(dtype) * y.abs() * (1 + 2.0 ** -8) + 2.0 ** -19 * size + 2.0 ** -25


def quantize(x):
    """(codes, scale, minimum) by the definition, fp32 arithmetic on the CPU: what the kernel has to give bit for bit."""

    dtype, x = x.dtype, x.detach().cpu().float()
    low, high = x.amin(-1), x.amax(-1)
    good = torch.isfinite(x).all(-1) & torch.isfinite(high - low)
    scale = ((high - low) / 15).to(dtype).float()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = ((x - low[..., None]) / scale[..., None]).round().clamp(max=15)
    codes = torch.where(good[..., None], codes, torch.zeros_like(codes)).to(torch.uint8)
    nan = torch.full_like(scale, math.nan)
    return codes, torch.where(good, scale, nan).to(dtype), torch.where(good, low, nan).to(dtype)


def pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def values(codes, params):
    """What cache entries stand for, in fp64."""

    return unpack(codes.cpu()).double() * params.cpu()[..., :1].double() + params.cpu()[..., 1:].double()


def attention(q, codes, params, table, seq_lens, query_starts=None, scale=None, window=None, rounded=None):
    """-> (result, bound): softmax attention in fp64, and how far the kernels' arithmetic may take each value; NaN for rows of no sequence.

    The bound adds up: the last rounding; the rounding of p * s (the probabilities times the value scales) to fp16 or, with ``rounded`` (a kernel
    that forms keys, values and probabilities in that type), of those three: independent errors of at most half a step h each, whose sum
    with weights a_i exceeds 7 h sqrt(sum a_i^2) with a probability below 2 exp(-49 / 2) = 5e-11 (Hoeffding); and fp32 sums, 2^-20 of the sum of
    the sizes (a score that is off by d moves the row by at most 2 d times the spread of its values)."""

    device = q.device
    pages, _, heads, page, _ = codes.shape
    tokens, q_heads, dim = q.shape
    each, batch = q_heads // heads, table.shape[0]
    table, lens = table.to(device), seq_lens.tolist()
    starts = list(range(batch + 1)) if query_starts is None else query_starts.tolist()
    scale = dim ** -0.5 if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=device)
    bound = torch.zeros_like(out)
    h, hp = half_step(q.dtype), half_step(rounded or torch.float16)
    for b in range(batch):
        n = min(max(lens[b], 0), table.shape[1] * page)
        q0 = min(max(starts[b], 0), tokens)
        m = min(max(starts[b + 1], q0), tokens) - q0
        if not m:
            continue
        at = torch.arange(n, device=device)
        ids = table[b][at // page].long()
        there = (ids >= 0) & (ids < pages)
        ids, rows = ids.clamp(0, max(pages - 1, 0)), at % page
        mine = n - m + torch.arange(m, device=device)[:, None]
        seen = there & (at <= mine)
        if window is not None:
            seen = seen & (at > mine - window)
        anything = seen.any(1)
        used = seen.any(0)
        seen, ids, rows = seen[:, used][:, None], ids[used], rows[used]
        for kh in range(heads):
            sl = slice(kh * each, (kh + 1) * each)
            (ks, km), (vs, vm) = (params[ids, i, kh, rows].to(device).double().unbind(-1) for i in (0, 1))
            (kc, vc) = (unpack(codes[ids, i, kh, rows].to(device)).double() for i in (0, 1))
            k, vc = kc * ks[:, None] + km[:, None], vc * vs[:, None]
            v = vc + vm[:, None]
            x = q[q0:q0 + m, sl].double()
            s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            p = s.softmax(-1) if len(ids) else s
            p = torch.where(anything[:, None, None] & seen, p, 0.0)
            y = p @ v
            out[q0:q0 + m, sl] = y
            spread = p @ v.abs() + y.abs()
            size = scale * x.abs().sum(-1, keepdim=True) * (15 * ks.abs() + km.abs()).max() if len(ids) else 0
            bad = 2 * 2.0 ** -20 * abs(size) * spread + 2.0 ** -20 * (p @ (vc.abs() + vm.abs()[:, None])) + h * y.abs() * (1 + 2.0 ** -6) + 2.0 ** -25
            weights = vc if rounded is None else torch.maximum(vc.abs(), v.abs())
            bad = bad + 7 * hp * (p.square() @ weights.square()).sqrt()
            if rounded is not None:
                # values (p_t v_t), and keys: a score's error has deviations of hp sqrt(sum (q k)^2) scale, which moves the row by p_t (v_t - y)
                moved = p.square() * (scale ** 2 * (x.square() @ k.square().T))
                second = (moved @ v.square() - 2 * y * (moved @ v) + y.square() * moved.sum(-1, keepdim=True)).clamp(min=0).sqrt()
                bad = bad + 7 * hp * ((p.square() @ v.square()).sqrt() + second)
            bound[q0:q0 + m, sl] = bad
    return out, bound
