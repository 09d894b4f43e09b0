"""What the operators beside the layers refuse, and the frequencies of the rotation: host logic, no GPU.  Arguments are checked before the device is looked at, so a call whose shapes are right
ends with the refusal of host memory."""
import ctypes
import math

import pytest
import torch

from hyperqwen_rtx4080s32_b200 import _lib, ops

E = _lib.GqError


def h(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def adapters(**new):
    s = dict(base=h(3, 24), x=h(3, 256), a=h(2, 16, 256), b=h(2, 24, 8), scales=h(2, 2, dtype=torch.float32), ids=h(3, dtype=torch.int64), n_outs=[16, 8], out=None)
    s.update(new)
    return ops.low_rank_add(**s)


@pytest.mark.parametrize("new,why", [
    ({}, "CUDA"), (dict(x=h(3, 256, dtype=torch.float16)), "x is bf16"), (dict(x=h(256)), "x is bf16"), (dict(x=h(3, 128)), "multiple of 256"), (dict(base=h(3, 25)), "base is"), (dict(base=h(4, 24)), "base is"),
    (dict(n_outs=[]), "one to eight"), (dict(n_outs=[3] * 9), "one to eight"), (dict(n_outs=[-8, 32]), "columns"), (dict(a=h(2, 24, 256)), "a is bf16"), (dict(a=h(3, 16, 256)), "a is bf16"),
    (dict(b=h(2, 24, 12), a=h(2, 24, 256)), "multiple of 8"), (dict(b=h(2, 24, 136), a=h(2, 272, 256)), "multiple of 8"), (dict(b=h(0, 24, 8), a=h(0, 16, 256)), "one adapter"), (dict(b=h(2, 23, 8)), "b is bf16"),
    (dict(a=h(2, 256, 16).transpose(1, 2)), "contiguous"), (dict(scales=h(2, 2)), "scales is"), (dict(scales=h(2, 1, dtype=torch.float32)), "scales is"), (dict(ids=h(2, dtype=torch.int64)), "ids is"),
    (dict(ids=h(3, dtype=torch.int16)), "ids is"), (dict(out=h(3, 23)), "out is"), (dict(out=h(24, 3).t()), "unit column stride"), (dict(out=h(1, 24).expand(3, 24)), "rows of their own")], ids=str)
def test_adapters(new, why):
    with pytest.raises(E, match=why):
        adapters(**new)


def heads(store=False, **new):
    s = dict(qkv=h(5, 8 * 16), positions=h(5, dtype=torch.int64), inv_freq=h(4, dtype=torch.float64), n_heads=4, n_kv_heads=2, head_dim=16)
    if store:
        s |= dict(k_pages=h(3, 4, 2, 16), v_pages=h(3, 4, 2, 16), slots=h(5, dtype=torch.int64))
    s.update(new)
    return (ops.qk_norm_rope_store if store else ops.qk_norm_rope)(**s)


@pytest.mark.parametrize("new,why", [
    ({}, "CUDA"), (dict(qkv=h(5, 120)), "qkv is"), (dict(qkv=h(5, 128, dtype=torch.float32)), "qkv is"), (dict(gated=True), "qkv is"), (dict(n_heads=0), "one or more"), (dict(n_kv_heads=0), "one or more"),
    (dict(head_dim=12), "multiple of 8"), (dict(head_dim=520), "multiple of 8"), (dict(head_dim=0), "multiple of 8"), (dict(positions=h(4, dtype=torch.int64)), "positions"), (dict(positions=h(5)), "positions"),
    (dict(inv_freq=h(4, dtype=torch.float32)), "inv_freq"), (dict(inv_freq=h(9, dtype=torch.float64)), "at most"), (dict(q_norm=h(15)), "norm weight"), (dict(k_norm=h(16, dtype=torch.float32)), "norm weight"),
    (dict(k_norm=h(32)[::2]), "contiguous")], ids=str)
def test_heads(new, why):
    with pytest.raises(E, match=why):
        heads(**new)


@pytest.mark.parametrize("new,why", [
    ({}, "CUDA"), (dict(k_pages=h(3, 4, 2, 8)), "k_pages is"), (dict(v_pages=h(3, 4, 1, 16)), "v_pages is"), (dict(v_pages=h(2, 4, 2, 16)), "same pages"), (dict(v_pages=h(3, 5, 2, 16)), "same pages"),
    (dict(k_pages=h(3, 0, 2, 16)), "one row"), (dict(k_pages=h(3, 4, 16, 2).transpose(2, 3)), "unit stride"), (dict(k_pages=h(3, 4, 2, 20)[..., :16]), "multiples of 16"),
    (dict(k_pages=h(1, 4, 2, 16).expand(3, 4, 2, 16)), "of its own"), (dict(slots=h(4, dtype=torch.int64)), "slots"), (dict(slots=h(5, dtype=torch.float32)), "slots")], ids=str)
def test_store(new, why):
    with pytest.raises(E, match=why):
        heads(store=True, **new)


def attend(**new):
    s = dict(q=h(4, 6, 64), k_pages=h(3, 16, 2, 64), v_pages=h(3, 16, 2, 64), page_table=h(2, 3, dtype=torch.int32), lens=h(2, dtype=torch.int32))
    s.update(new)
    return ops.paged_attention(**s)


@pytest.mark.parametrize("new,why", [
    ({}, "CUDA"), (dict(q=h(4, 6, 96)), "head_dim is"), (dict(q=h(4, 384)), "q is"), (dict(q=h(4, 6, 64, dtype=torch.float16)), "q is"), (dict(q=h(4, 5, 64)), "multiple of the key-value"), (dict(q=h(5, 6, 64)), "same number of tokens"),
    (dict(k_pages=h(3, 16, 2, 128)), "k_pages is"), (dict(v_pages=h(3, 16, 1, 64)), "v_pages is"), (dict(v_pages=h(4, 16, 2, 64)), "same pages"), (dict(k_pages=h(3, 16, 2, 72)[..., :64]), None),
    (dict(k_pages=h(3, 16, 2, 68)[..., :64]), "multiples of 16"), (dict(page_table=h(2, 3, dtype=torch.int64)), "page_table"), (dict(lens=h(2, dtype=torch.int64)), "lens"), (dict(lens=h(3, dtype=torch.int32)), "lens"),
    (dict(q_starts=h(2, dtype=torch.int32)), "q_starts"), (dict(gate=h(4, 6, 32)), "gate is"), (dict(gate=h(4, 64, 6).transpose(1, 2)), "unit stride"), (dict(out=h(4, 6, 64, dtype=torch.float32)), "out is"),
    (dict(out=h(1, 6, 64).expand(4, 6, 64)), "of their own"), (dict(page_table=h(0, 3, dtype=torch.int32), lens=h(0, dtype=torch.int32)), "same number")], ids=str)
def test_attention(new, why):
    with pytest.raises(E, match=why or "CUDA"):
        attend(**new)


def test_the_c_entries_refuse_what_they_cannot_take():
    L = _lib.lib()
    for name in ("gq_low_rank_add", "gq_head_norm_rope", "gq_paged_attention"):
        assert getattr(L, name)(None, None) == -3
    assert L.gq_low_rank_workspace_bytes(None) == -3 and L.gq_attention_workspace_bytes(None) == -3
    zeros = ctypes.create_string_buffer(1024)         # sizes of nothing: a shape that no call has
    for name in ("gq_low_rank_add", "gq_head_norm_rope", "gq_paged_attention"):
        assert getattr(L, name)(zeros, None) == -2


def test_frequencies():
    inv, amp = ops.rotary_frequencies(128, 1e6, device="cpu")
    assert inv.dtype == torch.float64 and inv.shape == (64,) and amp == 1.0
    assert all(math.isclose(float(v), 1e6 ** (-2 * i / 128), rel_tol=1e-14) for i, v in enumerate(inv))
    lin, amp = ops.rotary_frequencies(128, 1e6, scaling="linear", factor=4, device="cpu")
    assert torch.equal(lin, inv / 4) and amp == 1.0
    yarn, amp = ops.rotary_frequencies(128, 1e6, scaling="yarn", factor=4, original_context=32768, device="cpu")
    assert math.isclose(amp, 0.1 * math.log(4) + 1)
    turns = 32768 * inv / (2 * math.pi)                # pairs that turn often keep their frequency, those that turn less than once are divided
    assert torch.equal(yarn[turns > 40], inv[turns > 40]) and torch.allclose(yarn[turns < 0.8], inv[turns < 0.8] / 4, rtol=1e-12)
    assert bool(((yarn <= inv) & (yarn >= inv / 4 * (1 - 1e-12))).all()) and bool((yarn.diff() < 0).all())
    assert ops.rotary_frequencies(0, device="cpu")[0].numel() == 0
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, base=0), dict(rotary_dim=8, factor=-1), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="yarn", factor=2)):
        with pytest.raises(E):
            ops.rotary_frequencies(device="cpu", **bad)


def test_slots_of_a_cache():
    from hyperqwen_rtx4080s32_b200.attention import PagedKVCache

    cache = PagedKVCache(7, 4, 2, 8, device="cpu")
    assert cache.k.shape == cache.v.shape == (7, 4, 2, 8) and cache.k.stride() == (64, 8, 32, 1)
    table = torch.tensor([[5, 1], [6, 0]], dtype=torch.int32)
    got = cache.slots(table, torch.tensor([0, 0, 1, 1, 0]), torch.tensor([0, 6, 3, 4, -1]))
    assert got.tolist() == [20, 6, 27, 0, -1]
    for bad in ((0, 4), (4, 0)):
        with pytest.raises(E):
            PagedKVCache(*bad, 2, 8, device="cpu")


def test_heads_that_do_not_fit_the_projections():
    from hyperqwen_rtx4080s32_b200.attention import GGUFAttention
    from hyperqwen_rtx4080s32_b200.linear import GGUFLinear, LowRankAdapters

    inv = torch.zeros(4, dtype=torch.float64)
    o = GGUFLinear(512, [768])
    att = GGUFAttention(GGUFLinear(768, [1024, 128, 128]), o, 64, inv)
    assert att.gated and (att.n_heads, att.n_kv_heads) == (8, 2)
    assert not GGUFAttention(GGUFLinear(768, [512, 128, 128]), o, 64, inv).gated
    for rows in ([512, 128], [512, 128, 64], [768, 128, 128], [512, 96, 96]):
        with pytest.raises(E):
            GGUFAttention(GGUFLinear(768, rows), o, 64, inv)
    with pytest.raises(RuntimeError, match="no packed tiles"):
        LowRankAdapters(o, 2, 8)


def test_the_operators_trace_with_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    def fn(base, x, a, b, scales, ids, pos, inv, k_pages, v_pages, slots, table, lens):
        y = ops.low_rank_add(base, x, a, b, scales, ids, [64, 16, 16])
        q, _ = ops.qk_norm_rope(y, pos, inv, 4, 1, 16)
        q = ops.qk_norm_rope_store(y, pos, inv, 4, 1, 16, k_pages, v_pages, slots) + q
        return ops.paged_attention(q.repeat(1, 1, 4), k_pages.repeat(1, 1, 1, 4), v_pages.repeat(1, 1, 1, 4), table, lens)

    with FakeTensorMode():
        e = lambda *s, t=torch.bfloat16: torch.empty(s, dtype=t, device="meta")  # noqa: E731
        i64, i32 = torch.int64, torch.int32
        gm, _ = torch._dynamo.export(fn)(e(6, 96), e(6, 256), e(2, 24, 256), e(2, 96, 8), e(2, 3, t=torch.float32), e(6, t=i64), e(6, t=i64), e(8, t=torch.float64), e(3, 4, 1, 16),
                                         e(3, 4, 1, 16), e(6, t=i64), e(2, 2, t=i32), e(2, t=i32))
    names = str([n.target for n in gm.graph.nodes if n.op == "call_function"])
    assert all(n in names for n in ("low_rank_add", "qk_norm_rope", "qk_norm_rope_store", "paged_attention"))
