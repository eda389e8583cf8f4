"""What the operators between the projections refuse, and what their helpers build: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from attention_reference import pack, quantize, unpack, values
from conftest import seeded
from xqt_b200 import native
from xqt_b200.errors import XQTBackendError
from xqt_b200.ops.kv4 import allocate_kv4_cache, kv4_append, kv4_attention, kv4_gather
from xqt_b200.ops.rotary import _dense, qk_norm_rope, rotary_frequencies


def test_frequencies():
    f, axes = rotary_frequencies(8, theta=100.0)
    assert axes is None and torch.allclose(f, torch.tensor([1, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    f, axes = rotary_frequencies(12, theta=16.0, ladders=(4, 8))
    assert axes.tolist() == [0, 0, 1, 1, 1, 1] and torch.allclose(f, torch.tensor([1, 0.25, 1, 0.5, 0.25, 0.125], dtype=torch.float64))
    f, axes = rotary_frequencies(8, theta=16.0, sections=(1, 0, 3))
    assert axes.tolist() == [0, 2, 2, 2] and torch.allclose(f, torch.tensor([1, 0.5, 0.25, 0.125], dtype=torch.float64))


@pytest.mark.parametrize("args", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, sections=(1, 2)), dict(rotary_dim=8, ladders=(3, 5)),
                                  dict(rotary_dim=8, ladders=(4, 2)), dict(rotary_dim=8, sections=(4,), ladders=(8,)), dict(rotary_dim=8, theta=0.0),
                                  dict(rotary_dim=8, theta=float("inf")), dict(rotary_dim=8, sections=(5, -1))])
def test_frequencies_refused(args):
    with pytest.raises(XQTBackendError):
        rotary_frequencies(**args)


def _rope_call(**change):
    call = dict(q=torch.zeros(3, 4, 64, dtype=torch.float16), k=torch.zeros(3, 2, 64, dtype=torch.float16), positions=torch.arange(3),
                frequencies=rotary_frequencies(64)[0])
    call.update(change)
    return qk_norm_rope(call.pop("q"), call.pop("k"), call.pop("positions"), call.pop("frequencies"), **call)


@pytest.mark.parametrize("change,said", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros(3, 4, 64)), "fp16/bf16"), (dict(q=torch.zeros(3, 64, dtype=torch.float16)), "fp16/bf16"),
    (dict(q=torch.zeros(3, 4, 72, dtype=torch.float16)), "multiple of 16"), (dict(q=torch.zeros(3, 4, 272, dtype=torch.float16)), "multiple of 16"),
    (dict(q=torch.zeros(3, 0, 64, dtype=torch.float16)), "head"),
    (dict(k=torch.zeros(2, 2, 64, dtype=torch.float16)), "keys"), (dict(k=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "keys"),
    (dict(k=torch.zeros(3, 2, 32, dtype=torch.float16)), "keys"), (dict(k=None, k_weight=torch.ones(64)), "no keys"),
    (dict(frequencies=torch.ones(32)), "float64"), (dict(frequencies=torch.ones(36, dtype=torch.float64)), "multiple of 8"),
    (dict(frequencies=torch.ones(40, dtype=torch.float64)), "fit"), (dict(frequencies=torch.ones(64, dtype=torch.float64)[::2]), "contiguous"),
    (dict(positions=torch.arange(4)), "positions"), (dict(positions=torch.zeros(3)), "positions"), (dict(positions=torch.zeros((0, 3), dtype=torch.int64)), "axis"),
    (dict(axes=torch.zeros(32)), "axes"), (dict(axes=torch.zeros(31, dtype=torch.int32)), "axes"),
    (dict(q_weight=torch.ones(32)), "weights"), (dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=torch.float16)), "weights"),
    (dict(q_weight=torch.ones(64, dtype=torch.float64)), "weights"),
])
def test_rope_refusals(change, said):
    with pytest.raises(XQTBackendError, match=said):
        _rope_call(**change)


def test_shared_addresses_are_seen():
    x = torch.empty(4, 6, 32)
    assert _dense(x.shape, x.stride()) and _dense(x[:, :3].shape, x[:, :3].stride())
    y = x.transpose(0, 1)
    assert _dense(y.shape, y.stride())
    for z in (x[:1].expand(4, 6, 32), x[:, :1].expand(4, 6, 32), torch.empty(400).as_strided((4, 6, 32), (32, 32, 1)), x.transpose(1, 2)):
        assert not _dense(z.shape, z.stride())


def _attention_call(**change):
    codes, params = allocate_kv4_cache(5, 2, 64, page_size=16, dtype=torch.float16)
    call = dict(q=torch.zeros(3, 4, 64, dtype=torch.float16), codes=codes, params=params, block_table=torch.zeros(3, 2, dtype=torch.int32),
                seq_lens=torch.zeros(3, dtype=torch.int32))
    call.update(change)
    first = [call.pop(n) for n in ("q", "codes", "params", "block_table", "seq_lens")]
    return kv4_attention(*first, **call)


@pytest.mark.parametrize("change,said", [
    (dict(), "CUDA"),
    (dict(codes=torch.zeros(5, 2, 2, 16, 32)), "codes"), (dict(codes=torch.zeros(5, 1, 2, 16, 32, dtype=torch.uint8)), "codes"),
    (dict(codes=torch.zeros(5, 2, 2, 16, 48, dtype=torch.uint8)), "head dimension"), (dict(codes=torch.zeros(5, 2, 2, 8, 32, dtype=torch.uint8)), "page size"),
    (dict(codes=torch.zeros(5, 2, 2, 24, 32, dtype=torch.uint8)), "page size"), (dict(codes=torch.zeros(5, 2, 2, 16, 64, dtype=torch.uint8)[..., ::2]), "contiguous"),
    (dict(params=torch.zeros(5, 2, 2, 16, 2)), "params"), (dict(params=torch.zeros(5, 2, 2, 16, 1, dtype=torch.float16)), "params"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "queries"), (dict(q=torch.zeros(3, 3, 64, dtype=torch.float16)), "multiple"),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.float16)), "queries"), (dict(q=torch.zeros(4, 4, 64, dtype=torch.float16)), "one row"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int64)), "block table"), (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)[:, ::2]), "block table"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32)), "seq_lens"), (dict(seq_lens=torch.zeros(3, dtype=torch.int64)), "seq_lens"),
    (dict(query_starts=torch.zeros(3, dtype=torch.int32)), "query_starts"), (dict(query_starts=torch.zeros(4, dtype=torch.int64)), "query_starts"),
    (dict(window=0), "window"), (dict(scale=float("nan")), "scale"),
])
def test_attention_refusals(change, said):
    with pytest.raises(XQTBackendError, match=said):
        _attention_call(**change)


def test_append_and_gather_refusals():
    codes, params = allocate_kv4_cache(5, 2, 64, page_size=16, dtype=torch.float16)
    x, slots = torch.zeros(3, 2, 64, dtype=torch.float16), torch.arange(3)
    for k, v, s, said in ((x, x, slots, "CUDA"), (x, x[:2], slots, "keys and values"), (x.bfloat16(), x, slots, "keys and values"), (x, x, slots[:2], "keys and values"),
                          (x, x, slots.float(), "slots"), (x, x, torch.arange(6)[::2], "slots")):
        with pytest.raises(XQTBackendError, match=said):
            kv4_append(k, v, codes, params, s)
    with pytest.raises(XQTBackendError, match="CUDA"):
        kv4_gather(codes, params, slots)
    with pytest.raises(XQTBackendError, match="slots"):
        kv4_gather(codes, params, slots.float())
    for bad in (dict(head_dim=96), dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(kv_heads=0), dict(dtype=torch.float32), dict(pages=-1)):
        with pytest.raises(XQTBackendError):
            allocate_kv4_cache(**{**dict(pages=1, kv_heads=1, head_dim=64), **bad})


def test_entries_check_their_arguments_before_any_cuda_call():
    lib = native.library()
    steps = (ctypes.c_longlong * 10)()
    rope = lambda dim, rotary, tokens=1, q=16: lib.xqt_b200_qk_norm_rope(q, 0, 16, 0, 0, 0, 16, 16, 0, steps, tokens, 1, 0, dim, rotary, 1, 0, 0, 0, 2, 1e-6, 0)  # noqa: E731
    assert rope(24, 16) == 1 and rope(272, 16) == 1 and rope(64, 80) == 1 and rope(64, 24) == 1 and rope(64, 64, -1) == 1 and rope(64, 64, q=0) == 1
    assert rope(64, 64, q=8) == 1 and rope(64, 64, 0) == 0
    attend = lambda dim=64, page=16, each=1, tokens=1, width=1, pages=1, window=0, ws=0: lib.xqt_b200_kv4_attention(  # noqa: E731
        16, 16, 16, 16, 16, 0, 16, steps, tokens, 1, each, 1, dim, pages, page, width, window, 0, 1.0, ws, 0, 0, 0)
    assert attend(dim=96) == 1 and attend(page=8) == 1 and attend(page=24) == 1 and attend(page=8192) == 1 and attend(each=0) == 1
    assert attend(tokens=2) == 1 and attend(width=1 << 28) == 1 and attend(pages=1 << 31) == 1 and attend(window=-1) == 1 and attend(tokens=0) == 0
    append = lambda dim=64, tokens=1, heads=1: lib.xqt_b200_kv4_append(16, 8, 16, 16, 16, steps, tokens, heads, dim, 1, 16, 0, 0, 0)  # noqa: E731
    assert append(dim=96) == 1 and append(tokens=-1) == 1 and append(heads=0) == 1 and append() == 1 and append(tokens=0) == 0


def test_native_path_leaves_to_python_what_it_does_not_take():
    host = native.attention_host()
    codes, params = allocate_kv4_cache(2, 2, 64, page_size=16, dtype=torch.float16)
    x, slots = torch.zeros(3, 2, 64, dtype=torch.float16), torch.arange(3)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    assert host.kv4_append(x, x, codes, params, slots) is None and host.kv4_append(x, x) is None and host.kv4_append(None, x, codes, params, slots) is None
    assert host.kv4_gather(codes, params, slots) is None and host.kv4_gather(codes, 1, slots) is None
    assert host.kv4_attention(x, codes, params, table, lens, None, None, None, None) is None
    assert host.qk_norm_rope(x, None, slots, rotary_frequencies(64)[0], None, None, None, 1e-6, False) is None
    with pytest.raises(TypeError):
        host.qk_norm_rope(x, None, slots, rotary_frequencies(64)[0], None, None, None, "eps", False)


def test_definition_of_the_codes():
    x = torch.randn((7, 64), generator=seeded(1)).bfloat16()
    codes, scale, low = quantize(x)
    assert torch.equal(unpack(pack(codes)), codes)
    held = values(pack(codes), torch.stack((scale, low), -1))
    # half a step of the code, and at the top of the range what rounding the scale down (by at most 2^-8 of it) cuts off
    assert bool(((held - x.double()).abs() <= scale.double()[:, None] * (0.5 + 15 * 2.0 ** -8)).all())
