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


def long_prompt(keys, dim, dtype, queries, exponent=None, seed=81):
    """A key head per SM, so that every one has whole items; the tables go round 64 pages.  Values lie in [0.53, 1.47] with a mean of 1.  With ``exponent`` the first key is
    2 ** exponent times as probable as the others are on average, and its values are 0.  -> arguments, and those of the first two heads for the reference."""

    heads = torch.cuda.get_device_properties(0).multi_processor_count
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
