"""Guards of the operators beside the layers that need no GPU: the order of programmatic launches, refusals, files and banks."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

from hyperqwen_rtx4080s32_b200 import _lib, loader, ops
from hyperqwen_rtx4080s32_b200.attention import GGUFAttention, PagedKVCache
from hyperqwen_rtx4080s32_b200.linear import GGUFLinear, GGUFLinearMethod, LowRankAdapters

import test_block_ops_cpu as refusals

E, h = ops.GqError, refusals.h
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hyperqwen-rtx4080s32_b200", "csrc")


def kernels(text):
    """(name, body) of every __global__ function with a body, comments left out."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__", text):
        at = text.index("{", m.end())
        name = re.search(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", text[m.end():at])).group(1)
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield name, text[at:end]


@pytest.mark.parametrize("header", ["gq_adapters.cuh", "gq_heads.cuh", "gq_paged.cuh"])
def test_every_kernel_waits_for_the_one_in_front_on_every_path(header):
    """These kernels are launched programmatically, and some let the next one start at once.  A kernel that ends without the wait may end before the
    kernel in front of it does, and what is launched behind it waits for it alone: so the wait stands in front of the first return, and in no branch."""
    with open(os.path.join(CSRC, header), encoding="utf-8") as f:
        found = list(kernels(f.read()))
    assert found
    for name, body in found:
        assert body.count("pdl_wait();") == 1, name
        ahead = body[:body.index("pdl_wait();")]
        assert "return" not in ahead, f"{name} returns before it has waited"
        assert ahead.count("{") - ahead.count("}") == 1 and ahead.rstrip()[-1] in ";}", f"{name} waits in a branch"


@pytest.mark.parametrize("missing", [("k_pages",), ("v_pages",), ("slots",), ("k_pages", "slots"), ("k_pages", "v_pages", "slots")], ids=str)
def test_a_store_without_a_part_of_its_cache_is_refused(missing):
    with pytest.raises(E, match="all given"):
        refusals.heads(store=True, **{name: None for name in missing})


K = 256


def write_gguf(path, tensors, arch="qwen35", **meta):
    from gguf import GGUFWriter

    w = GGUFWriter(str(path), arch)
    for key, v in meta.items():
        key = key.replace("__", ".")
        (w.add_string if isinstance(v, str) else w.add_float32 if isinstance(v, float) else w.add_uint32)(key, v)
    for name, arr in tensors:
        w.add_tensor(name, arr)
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    return str(path)


def loaded_layer(n_outs, ids, k=K):
    """What LowRankAdapters looks at of a layer, in host memory."""
    lin = torch.nn.Module()
    lin.weight = torch.nn.Module()
    lin.weight.shard_id = list(ids)
    lin.gguf_tiles = {sid: None for sid in ids}
    lin.gguf_tiles_rows = dict(zip(ids, n_outs))
    lin.gguf_groups = {ids[0]: (torch.zeros(1, dtype=torch.uint8), None, None, list(ids), k // 256, 0)}
    return lin


def model_with_banks(slots=3, rank=8):
    model = loader.LoadedModel()
    for key, n_outs, ids in (("layers.3.self_attn.qkv_proj", (48, 16, 16), ("q", "k", "v")), ("layers.3.self_attn.o_proj", (24,), (None,))):
        lin = model.linears[key] = loaded_layer(n_outs, ids)
        bank = lin.gguf_adapters = LowRankAdapters(lin, slots, rank)
        for t in (bank.a, bank.b, bank.scales):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(t.numel())))
    return model


def pair(name, r, n_out, k=K):
    return [(f"{name}.lora_a", np.ones((r, k), np.float32)), (f"{name}.lora_b", np.ones((n_out, r), np.float32))]


GOOD = pair("blk.3.attn_q.weight", 4, 48)


@pytest.mark.parametrize("slot,tensors", [
    (0, GOOD + pair("blk.3.attn_output.weight", 4, 24, k=512)), (0, GOOD + pair("blk.3.attn_output.weight", 4, 32)), (0, GOOD + pair("blk.3.attn_k.weight", 4, 48)),
    (0, GOOD + [pair("blk.3.attn_v.weight", 4, 16)[0], pair("blk.3.attn_v.weight", 5, 16)[1]]), (0, GOOD + [("blk.3.attn_v.weight.lora_a", np.ones(K, np.float32)), pair("blk.3.attn_v.weight", 1, 16)[1]]),
    (-1, GOOD), (3, GOOD), (-1, []), (3, [])], ids=["K", "rows", "another shard's rows", "two ranks", "a row", "slot -1", "slot 3", "nothing into slot -1", "nothing into slot 3"])
def test_an_adapter_that_does_not_fit_changes_nothing(tmp_path, slot, tensors):
    model = model_with_banks()
    banks = [lin.gguf_adapters for lin in model.linears.values()]
    before = [t.clone() for b in banks for t in (b.a, b.b, b.scales)]
    path = write_gguf(tmp_path / "adapter.gguf", tensors, general__type="adapter", adapter__type="lora", adapter__lora__alpha=8.0)
    with pytest.raises((E, ValueError)):
        loader.load_adapter(path, model, slot)
    assert all(torch.equal(t, old) for t, old in zip([t for b in banks for t in (b.a, b.b, b.scales)], before))


def test_an_adapter_that_fits_fills_its_slot_alone(tmp_path):
    model = model_with_banks()
    bank, other = (lin.gguf_adapters for lin in model.linears.values())
    before = [bank.a.clone(), bank.b.clone()]
    path = write_gguf(tmp_path / "adapter.gguf", GOOD, general__type="adapter", adapter__type="lora", adapter__lora__alpha=8.0)
    assert loader.load_adapter(path, model, 1, scale=0.5) == ["layers.3.self_attn.qkv_proj"]
    assert bool((bank.a[1, :4] == 1).all()) and not bool(bank.a[1, 4:].any()) and bool((bank.b[1, :48, :4] == 1).all()) and not bool(bank.b[1, 48:].any()) and not bool(bank.b[1, :, 4:].any())
    assert bank.scales[1].tolist() == [1.0, 0.0, 0.0] and not bool(other.a[1].any()) and not bool(other.scales[1].any())
    assert torch.equal(bank.a[[0, 2]], before[0][[0, 2]]) and torch.equal(bank.b[[0, 2]], before[1][[0, 2]])
    for slot in (-1, 3):
        with pytest.raises(E, match="no slot"):
            bank.clear(slot)


def test_heads_that_the_attention_does_not_take_are_refused_when_the_block_is_made():
    inv = torch.zeros(4, dtype=torch.float64)
    for d in (64, 128, 256):
        assert GGUFAttention(GGUFLinear(512, [6 * d, 2 * d, 2 * d]), GGUFLinear(6 * d, [512]), d, inv).n_heads == 6
    for d in (96, 32, 16, 512, 8):
        with pytest.raises(E, match="attention takes heads of"):
            GGUFAttention(GGUFLinear(512, [8 * d, 2 * d, 2 * d]), GGUFLinear(8 * d, [512]), d, inv)
    for n_heads, n_kv in ((5, 2), (2, 4), (4, 0)):
        with pytest.raises(E, match="do not fit"):
            GGUFAttention(GGUFLinear(512, [n_heads * 64, n_kv * 64, n_kv * 64]), GGUFLinear(n_heads * 64, [512]), 64, inv)


@pytest.mark.parametrize("call,names", [(refusals.adapters, dict(x=(3, 256), base=(3, 24), b=(2, 24, 8))), (refusals.heads, dict(qkv=(5, 128))), (refusals.attend, dict(q=(4, 6, 64), v_pages=(3, 16, 2, 64)))], ids=["adapters", "heads", "attention"])
def test_a_forward_tangent_is_refused(call, names):
    import torch.autograd.forward_ad as fwd

    for name, shape in names.items():
        with fwd.dual_level(), pytest.raises(E, match="forward derivative"):
            call(**{name: fwd.make_dual(h(*shape), h(*shape))})


class HeadNormArgs(ctypes.Structure):
    """gq_head_norm_args of include/gq_b200.h."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("qkv", "positions", "inv_freq", "q_norm", "k_norm", "q_out", "k_out", "k_pages", "v_pages", "slots")] + [
        (n, ctypes.c_int64) for n in ("T", "ld_qkv", "n_pages")] + [("k_strides", ctypes.c_int64 * 3), ("v_strides", ctypes.c_int64 * 3)] + [
        (n, ctypes.c_int32) for n in ("n_heads", "n_kv_heads", "head_dim", "rotary_dim", "page_size", "positions_bytes", "slots_bytes", "interleaved", "gated")] + [("eps", ctypes.c_float), ("amplitude", ctypes.c_float)]


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are none: what is accepted has to end at the missing device")
@pytest.mark.parametrize("pages,slots,k_out,n_pages,accepted", [
    (False, True, False, 0, True), (False, True, False, 3, False), (True, True, False, 3, True), (True, False, False, 3, False), (True, True, True, 3, False), (False, False, True, 0, True),
    (False, True, True, 0, True), (False, False, False, 0, False)], ids=str)
def test_what_says_that_keys_are_stored(pages, slots, k_out, n_pages, accepted):
    """Pages, or slots without an output for keys: a cache of no pages has null pointers and is stored into all the same (no slot is inside it)."""
    a = HeadNormArgs(T=2, ld_qkv=256, n_pages=n_pages, n_heads=2, n_kv_heads=1, head_dim=64, page_size=16, positions_bytes=8, slots_bytes=8)
    a.qkv = a.q_out = a.positions = 1 << 20
    if pages:
        a.k_pages = a.v_pages = 1 << 20
    a.slots, a.k_out = (1 << 20) if slots else None, (1 << 20) if k_out else None
    assert (_lib.lib().gq_head_norm_rope(ctypes.byref(a), None) == -3) == (not accepted)


def test_the_status_message_names_what_the_word_reports(monkeypatch):
    lin = GGUFLinear(256, [64])
    assert isinstance(lin.quant_method, GGUFLinearMethod)
    monkeypatch.setattr(ops, "device_status", lambda device=None, clear=True: 2)
    with pytest.raises(RuntimeError, match="status 2") as raised:
        lin.quant_method.check_status()
    assert all(cause in str(raised.value) for cause in ("shape", "type", "embedding", "adapters", "slot", "page outside a cache", "page table"))
    monkeypatch.setattr(ops, "device_status", lambda device=None, clear=True: 0)
    lin.quant_method.check_status()


def test_slots_where_the_table_has_no_page():
    cache = PagedKVCache(7, 4, 2, 8, device="cpu")
    table = torch.tensor([[5, 1], [6, -1], [7, 0]], dtype=torch.int32)
    seqs, positions = torch.tensor([0, 0, 1, 1, 2, 2, 3, -1, 3, 0]), torch.tensor([7, 8, 3, 4, 0, 4, 0, 0, -1, 1 << 40])
    assert cache.slots(table, seqs, positions).tolist() == [7, 28, 27, 28, 28, 0, 28, 28, -1, 28]
    for empty in (table[:0], table[:, :0]):
        got = cache.slots(empty, torch.tensor([0, 0]), torch.tensor([0, -1]))
        assert got.dtype == torch.int64 and got.tolist() == [28, -1]


def test_outputs_and_caches_whose_own_parts_share_memory_are_refused():
    buf = h(4096)
    for strides in ((64, 64, 1), (64, 128, 1), (128, 64, 1), (320, 64, 1)):       # heads or tokens that begin inside another's
        with pytest.raises(E, match="of their own"):
            refusals.attend(out=buf.as_strided((4, 6, 64), strides))
    for strides in ((384, 64, 1), (64, 256, 1), (72, 300, 1)):
        with pytest.raises(E, match="CUDA"):
            refusals.attend(out=buf.as_strided((4, 6, 64), strides))
    for strides in ((32, 32, 16, 1), (128, 16, 16, 1), (64, 32, 16, 1)):
        with pytest.raises(E, match="of their own"):
            refusals.heads(store=True, k_pages=buf.as_strided((3, 4, 2, 16), strides))


def test_keys_and_values_in_one_memory_are_refused_and_side_by_side_are_not():
    one = h(3, 4, 2, 16)
    buf, both = h(4, 4, 2, 16), h(3, 2, 4, 2, 16)
    for k, v in ((one, one), (buf[:3], buf[1:]), (buf[1:], buf[:3])):
        with pytest.raises(E, match="pages of their own"):
            refusals.heads(store=True, k_pages=k, v_pages=v)
    flat, by_head, turns = h(3, 4, 4, 16), h(3, 2, 8, 16), h(6, 4, 2, 16)
    for k, v in ((both[:, 0], both[:, 1]), (both[:, 1], both[:, 0]), (flat[:, :, :2], flat[:, :, 2:]), (flat[:, :, ::2], flat[:, :, 1::2]), (by_head[:, :, :4].transpose(1, 2), by_head[:, :, 4:].transpose(1, 2)),
                 (turns[::2], turns[1::2]), (one, one.clone())):
        with pytest.raises(E, match="CUDA"):
            refusals.heads(store=True, k_pages=k, v_pages=v)
    rows = h(800)
    with pytest.raises(E, match="pages of their own"):                   # a row further: most rows are shared
        refusals.heads(store=True, k_pages=rows.as_strided((3, 4, 2, 16), (128, 32, 16, 1)), v_pages=rows.as_strided((3, 4, 2, 16), (128, 32, 16, 1), 32))


@pytest.mark.parametrize("x_shape,residual_shape", [((2, 3, K), (2, 3, K)), ((2, 3, K), (6, K)), ((6, K), (6, K)), ((6, K), (2, 3, K))], ids=str)
def test_a_residual_of_any_shape_in_front_of_a_layer_with_adapters(monkeypatch, x_shape, residual_shape):
    """As in front of the layer alone: the rows are what counts, and residual_out comes back as rows."""
    lin, seen = loaded_layer((24,), (None,)), []
    method = GGUFLinear(K, [24]).quant_method
    bank = lin.gguf_adapters = LowRankAdapters(lin, 2, 8)
    monkeypatch.setattr(method, "apply", lambda layer, x, bias=None: x[..., :24].clone())
    monkeypatch.setattr(bank, "add_", lambda y, x, ids: seen.append((x, ids)) or y)
    g = torch.Generator().manual_seed(1)
    x, residual = (torch.randn(s, generator=g).to(torch.bfloat16) for s in (x_shape, residual_shape))
    pre = ops.PreAddRMSNorm(torch.ones(K, dtype=torch.bfloat16), residual=residual)
    ids = torch.zeros(x_shape[:-1], dtype=torch.int64)
    out = method.apply_with_adapters(lin, x, ids, pre)
    plain = ops.PreAddRMSNorm(torch.ones(K, dtype=torch.bfloat16), residual=residual.reshape(-1, K))
    want = plain.unfused(x.reshape(-1, K))
    assert out.shape == (*x_shape[:-1], 24) and torch.equal(out.reshape(-1, 24), want[:, :24]) and torch.equal(seen[0][0].reshape(-1, K), want)
    assert torch.equal(pre.residual_out.reshape(-1, K), plain.residual_out) and pre.residual_out.shape == (6, K)


def block_model(d=64, unmapped=(), **meta):
    """A loaded model of one attention block in host memory, its file's numbers under `meta` (rope__scaling__type for "rope.scaling.type")."""
    model = loader.LoadedModel(meta={k.replace("__", "."): v for k, v in meta.items()}, unmapped=list(unmapped))
    for key, lin in (("layers.3.self_attn.qkv_proj", GGUFLinear(512, [8 * d, 2 * d, 2 * d])), ("layers.3.self_attn.o_proj", GGUFLinear(8 * d, [512]))):
        lin.gguf_groups = {"q": (torch.zeros(1, dtype=torch.uint8),)}
        model.linears[key] = lin
    return model


def test_the_files_scaling_is_taken_whole():
    meta = dict(rope__freq_base=1e6, rope__scaling__type="yarn", rope__scaling__factor=4.0, rope__scaling__original_context_length=4096, attention__key_length=64)
    want = ops.rotary_frequencies(64, 1e6, scaling="yarn", factor=4.0, original_context=4096, beta_fast=16.0, beta_slow=2.0, device="cpu")
    got = block_model(rope__scaling__yarn_beta_fast=16.0, rope__scaling__yarn_beta_slow=2.0, rope__scaling__yarn_ext_factor=1.0, **meta).attention(3)
    assert torch.equal(got.inv_freq, want[0]) and got.amplitude == want[1]
    usual = block_model(**meta).attention(3)
    assert torch.equal(usual.inv_freq, ops.rotary_frequencies(64, 1e6, scaling="yarn", factor=4.0, original_context=4096, device="cpu")[0]) and not torch.equal(usual.inv_freq, got.inv_freq)
    assert torch.equal(block_model(**meta).attention(3, beta_fast=16.0, beta_slow=2.0).inv_freq, want[0])


@pytest.mark.parametrize("meta,unmapped", [
    (dict(rope__scaling__attn_factor=1.2), ()), (dict(rope__scaling__yarn_attn_factor=0.9), ()), (dict(rope__scaling__yarn_ext_factor=0.5), ()), (dict(rope__scaling__yarn_log_multiplier=0.1), ()),
    (dict(rope__scaling__alpha=1000.0), ()), (dict(rope__scaling__factor=8.0), ()), ({}, ("rope_freqs.weight",)), ({}, ("blk.3.rope_factors_long.weight",))], ids=str)
def test_scaling_that_is_not_known_is_refused(meta, unmapped):
    model = block_model(attention__key_length=64, unmapped=unmapped, **meta)
    with pytest.raises(ValueError, match="does not do"):
        model.attention(3)
    assert torch.equal(model.attention(3, scaling="linear", factor=2.0).inv_freq, ops.rotary_frequencies(64, scaling="linear", factor=2.0, device="cpu")[0])


@pytest.mark.parametrize("meta", [dict(attention__sliding_window=4096), dict(attention__scale=0.1), dict(attn_logit_softcapping=50.0), dict(attention__max_alibi_bias=8.0), dict(attention__clamp_kqv=8.0),
                                  dict(attention__causal=False)], ids=str)
def test_an_attention_of_another_kind_is_refused(meta):
    with pytest.raises(ValueError, match="does not do"):
        block_model(attention__key_length=64, **meta).attention(3, scaling="none")
    assert block_model(attention__key_length=64, attention__sliding_window=0, attention__causal=True).attention(3).n_heads == 8


@pytest.mark.parametrize("bad", [dict(base=1.0), dict(base=0.5), dict(beta_slow=0.0), dict(beta_fast=0.0), dict(beta_slow=-1.0), dict(beta_slow=40.0), dict(beta_fast=float("inf")), dict(base=float("nan")), dict(factor=float("nan")),
                                 dict(factor=float("inf")), dict(base=float("inf")), dict(original_context=float("nan")), dict(original_context=-4)], ids=str)
def test_rotations_that_are_none_are_refused(bad):
    with pytest.raises(E):
        ops.rotary_frequencies(**{**dict(rotary_dim=64, base=1e4, scaling="yarn", factor=4.0, original_context=4096), **bad}, device="cpu")


def test_trained_parameters_are_loaded_as_values():
    bank = LowRankAdapters(loaded_layer((24,), (None,)), 2, 8)
    a, b = (torch.nn.Parameter(torch.ones(s)) for s in ((4, K), (24, 4)))
    bank.load(1, a, b, torch.tensor(0.5))
    assert not any(t.requires_grad for t in (bank.a, bank.b, bank.scales)) and a.requires_grad
    assert bool((bank.a[1, :4] == 1).all()) and bool((bank.b[1, :, :4] == 1).all()) and bank.scales[1, 0] == 0.5


class AttentionArgs(ctypes.Structure):
    """gq_attention_args of include/gq_b200.h."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k_pages", "v_pages", "page_table", "lens", "q_starts", "gate", "out")] + [(n, ctypes.c_int64) for n in ("T", "n_seqs", "table_width", "ld_table", "n_pages")] + [
        (n, ctypes.c_int64 * 2) for n in ("q_strides", "gate_strides", "out_strides")] + [(n, ctypes.c_int64 * 3) for n in ("k_strides", "v_strides")] + [
        (n, ctypes.c_int32) for n in ("n_heads", "n_kv_heads", "head_dim", "page_size")] + [("scale", ctypes.c_float), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)]


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are none: what is accepted has to end at the missing device")
@pytest.mark.parametrize("which", ["k_strides", "v_strides"])
@pytest.mark.parametrize("strides,accepted", [((2048, 64, 1024), True), ((0, 64, 0), True), ((-2048, 64, 1024), False), ((2048, -64, 1024), False), ((2048, 64, -1024), False), ((2048, 60, 1024), False)], ids=str)
def test_strides_of_pages_at_the_c_entries(which, strides, accepted):
    """A negative stride between rows would be taken as 32 unsigned bits, and one that leads below the first page as a slot that is none."""
    at = 1 << 20
    a = AttentionArgs(q=at, k_pages=at, v_pages=at, page_table=at, lens=at, out=at, T=2, n_seqs=2, table_width=4, ld_table=4, n_pages=8, n_heads=2, n_kv_heads=2, head_dim=64, page_size=16, scale=1.0)
    b = HeadNormArgs(qkv=at, q_out=at, positions=at, slots=at, k_pages=at, v_pages=at, T=2, ld_qkv=384, n_pages=8, n_heads=2, n_kv_heads=2, head_dim=64, page_size=16, positions_bytes=8, slots_bytes=8)
    for args, entry in ((a, "gq_paged_attention"), (b, "gq_head_norm_rope")):
        args.k_strides[:] = args.v_strides[:] = (2048, 64, 1024)
        getattr(args, which)[:] = strides
        assert (getattr(_lib.lib(), entry)(ctypes.byref(args), None) == -3) == (not accepted)
