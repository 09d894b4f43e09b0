"""The operators beside the quantized layers together: adapters beside a loaded layer, the attention half of a block through prompts, decode and
verification, and both from GGUF files."""
import numpy as np
import pytest
import torch

from hyperqwen_rtx4080s32_b200 import formats as F
from hyperqwen_rtx4080s32_b200 import loader, ops, synth
from hyperqwen_rtx4080s32_b200.attention import GGUFAttention, PagedKVCache
from hyperqwen_rtx4080s32_b200.linear import GGUFLinear

import test_gpu_adapters as adapters
import test_gpu_paged as paged


pytestmark = pytest.mark.gpu


def layer(k, rows, types, seed=0):
    lin = GGUFLinear(k, list(rows))
    ids = [None] if len(rows) == 1 else [0, 1] if len(rows) == 2 else ["q", "k", "v"]
    for i, (n, t, sid) in enumerate(zip(rows, types, ids)):
        lin.load_shard(synth.random_blocks(n, k, t, seed=seed + i, device="cuda"), t, sid)
    return lin.finalize()


def fill(lin, n_adapters, rank, seed=0):
    """A bank of adapters of different ranks, the last slot empty; returns it."""
    bank = lin.quant_method.add_adapters(lin, n_adapters, rank)
    for slot in range(n_adapters - 1):
        for j, (sid, n) in enumerate(zip(bank.order, bank.n_outs)):
            r = max(1, rank - 3 * slot - j)
            bank.load(slot, adapters.bf16(r, bank.k, seed=seed + 10 * slot + j, std=bank.k ** -0.5).float(), adapters.bf16(n, r, seed=seed + 500 + 10 * slot + j).half(), 0.5 + slot, sid)
    return bank


@pytest.mark.parametrize("rows,types", [((320,), (F.Q4_K,)), ((256, 64, 72), (F.Q4_K, F.Q4_K, F.Q4_K)), ((256, 64, 64), (F.IQ3_S, F.Q4_K, F.Q6_K)), ((200, 130), (F.Q8_0, F.IQ2_XS))], ids=str)
@pytest.mark.parametrize("m", [1, 9, 40, 150])
def test_a_layer_with_adapters(rows, types, m):
    lin = layer(1024, rows, types)
    bank = fill(lin, 4, 16)
    assert bank.n_outs == list(rows) and bank.a.shape == (4, len(rows) * 16, 1024)
    x, ids = synth.activations(m, 1024, device="cuda"), torch.arange(m, device="cuda") % 5 - 1
    base = lin(x)
    s = dict(base=base, x=x, a=bank.a, b=bank.b, scales=bank.scales, ids=ids, n_outs=bank.n_outs)
    got = lin(x, adapters=ids)
    assert torch.equal(got, adapters.call(s))
    adapters.check(got, s)
    assert torch.equal(got[ids == -1], base[ids == -1]) and torch.equal(got[ids == 3], base[ids == 3])        # none, and an empty slot
    assert torch.equal(lin(x.view(1, m, 1024), adapters=ids.int()), got.view(1, m, -1))
    for pre, wide in ((ops.PreSiluMul(), synth.activations(m, 2048, device="cuda")), (ops.PreAddRMSNorm(torch.ones(1024, dtype=torch.bfloat16, device="cuda"), residual=x.clone()), x)):
        assert torch.equal(lin(wide, pre=pre, adapters=ids), lin(pre.unfused(wide), adapters=ids))
    bank.clear(0)
    assert torch.equal(lin(x, adapters=torch.zeros_like(ids)), base)
    assert ops.device_status() == 0


def test_adapters_that_do_not_fit_are_refused():
    lin = layer(512, (64, 32), (F.Q4_K, F.Q6_K))
    x = synth.activations(2, 512, device="cuda")
    ids = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="add_adapters"):
        lin(x, adapters=ids)
    bank = lin.quant_method.add_adapters(lin, 2, 5)
    assert bank.rank == 8
    a, b = torch.zeros(5, 512), torch.zeros(64, 5)
    for bad in (dict(slot=2), dict(shard_id=7), dict(a=torch.zeros(5, 256)), dict(b=torch.zeros(32, 5)), dict(b=torch.zeros(64, 4)), dict(a=torch.zeros(9, 512), b=torch.zeros(64, 9))):
        with pytest.raises(ops.GqError):
            bank.load(**{**dict(slot=0, a=a, b=b, scale=1.0, shard_id=0), **bad})
    for n, r in ((0, 8), (1, 0), (1, 129)):
        with pytest.raises(ops.GqError):
            lin.quant_method.add_adapters(lin, n, r)
    with pytest.raises(ops.GqError, match="sum over the ranks"), ops.fused_allreduce(object()):
        lin(x, adapters=ids)


def block(gated, hidden=768, hq=6, hk=2, d=64, rot=32):
    qkv = layer(hidden, ((2 if gated else 1) * hq * d, hk * d, hk * d), (F.Q4_K, F.IQ3_S, F.Q6_K), seed=20)
    o = layer(hq * d if hq * d % 256 == 0 else 512, (hidden,), (F.IQ4_XS,), seed=40)
    inv, amp = ops.rotary_frequencies(rot, 1e6)
    return GGUFAttention(qkv, o, d, inv, amplitude=amp, q_norm=1 + adapters.bf16(d, seed=1, std=0.1), k_norm=1 + adapters.bf16(d, seed=2, std=0.1))


@pytest.mark.parametrize("gated,with_adapters", [(False, True), (True, False), (True, True)])
def test_prompts_decode_and_verification_through_a_block(gated, with_adapters):
    """Every stage against its definition, on what the stage before it left: the cache's rows, the attention, the whole call."""
    att = block(gated, hq=8, hk=2)
    if with_adapters:
        fill(att.qkv, 3, 8)
        fill(att.o, 3, 16, seed=7)
    cache, width = att.cache(40, 16), 12
    table = torch.randperm(40, generator=torch.Generator().manual_seed(3))[:3 * width].view(3, width).int().cuda()
    have = torch.zeros(3, dtype=torch.int64)
    filled = torch.zeros(40 * 16, dtype=torch.bool, device="cuda")
    for step, news in enumerate(([37, 5, 90], [1, 1, 1], [1, 1, 1], [4, 4, 4], [3, 0, 2], [1, 1, 1])):
        t = sum(news)
        x = synth.activations(t, 768, seed=step, device="cuda")
        seqs = torch.tensor([b for b, n in enumerate(news) for _ in range(n)], device="cuda")
        positions = torch.cat([torch.arange(int(have[b]), int(have[b]) + n) for b, n in enumerate(news)]).cuda()
        have += torch.tensor(news)
        lens = have.int().cuda()
        slots = cache.slots(table, seqs, positions)
        starts = None if len(set(news)) == 1 else torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32, device="cuda")
        ids = seqs - 1 if with_adapters else None
        before = [cache.k.clone(), cache.v.clone()]
        got = att(x, positions, cache, slots, table, lens, q_starts=starts, adapters=ids)
        # what the layer leaves, stage by stage
        qkv = att.qkv(x, adapters=ids)
        how = dict(q_norm=att.q_norm, k_norm=att.k_norm, eps=att.eps, amplitude=att.amplitude, gated=gated)
        q, k = ops.qk_norm_rope(qkv, positions, att.inv_freq, 8, 2, 64, **how)
        v = qkv[:, -128:].reshape(t, 2, 64)
        filled[slots] = True
        for pages, old, new in ((cache.k, before[0], k), (cache.v, before[1], v)):
            old = old.reshape(-1, 2, 64)
            old[slots] = new
            assert torch.equal(pages.reshape(-1, 2, 64), old)
        gate = qkv[:, :16 * 64].view(t, 8, 128)[..., 64:] if gated else None
        more = dict(q_starts=starts, gate=gate)
        s = dict(q=q, k_pages=cache.k, v_pages=cache.v, page_table=table, lens=lens)
        out = ops.paged_attention(**s, **more)
        paged.check(out, s, more, [0] + list(np.cumsum(news)))
        assert torch.equal(got, att.o(out.flatten(1), adapters=ids))
    assert not bool(cache.k.reshape(-1, 128)[~filled].any())
    assert ops.device_status() == 0


def test_a_decode_step_captured_with_padding():
    """A graph of a fixed batch: fewer sequences than rows leave length 0, no slot and no adapter; replayed as the sequences grow."""
    att = block(True, hq=8, hk=2)
    fill(att.qkv, 2, 8)
    fill(att.o, 2, 8)
    b, width = 5, 6
    cache, eager = att.cache(b * width, 16), att.cache(b * width, 16)
    table = torch.arange(b * width, device="cuda").view(b, width).int()
    x, positions = synth.activations(b, 768, device="cuda"), torch.full((b,), -1, device="cuda")
    slots, lens, ids = torch.full((b,), -1, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda"), torch.full((b,), -1, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        att(x, positions, cache, slots, table, lens, adapters=ids)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        out = att(x, positions, cache, slots, table, lens, adapters=ids)
    for step in range(40):
        live = 1 + step // 10                     # sequences come in one by one
        x.copy_(synth.activations(b, 768, seed=step, device="cuda"))
        pos = torch.tensor([step - 10 * i if i < live else -1 for i in range(b)], device="cuda")
        positions.copy_(pos)
        slots.copy_(cache.slots(table, torch.arange(b, device="cuda"), pos))
        lens.copy_((pos + 1).int())
        ids.copy_(torch.where(pos < 0, -1, torch.arange(b, device="cuda") % 2))
        graph.replay()
        want = att(x, positions, eager, slots, table, lens, adapters=ids)
        assert torch.equal(out, want) and torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v)
    assert ops.device_status() == 0


def _write(path, tensors, arch="qwen35", **meta):
    from gguf import GGMLQuantizationType, GGUFWriter

    w = GGUFWriter(path, arch)
    for key, v in meta.items():
        key = key.replace("__", ".")
        (w.add_string if isinstance(v, str) else w.add_float32 if isinstance(v, float) else w.add_uint32)(key, v)
    for name, arr, t in tensors:
        w.add_tensor(name, arr) if t is None else w.add_tensor(name, arr, raw_dtype=GGMLQuantizationType(t))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()


def test_a_block_and_its_adapter_from_files(tmp_path):
    k, d, rng = 512, 64, np.random.default_rng(5)
    spec = [("attn_q", 2 * 512, k, F.Q4_K), ("attn_k", 128, k, F.Q4_K), ("attn_v", 128, k, F.Q4_K), ("attn_output", k, 512, F.IQ4_XS), ("ffn_gate", 768, k, F.Q4_K), ("ffn_up", 768, k, F.Q6_K)]
    tensors = [(f"blk.3.{n}.weight", synth.random_blocks(no, kk, t, seed=i).numpy(), t) for i, (n, no, kk, t) in enumerate(spec)]
    norms = {n: (1 + 0.1 * rng.standard_normal(d)).astype(np.float32) for n in ("q", "k")}
    tensors += [(f"blk.3.attn_{n}_norm.weight", w, None) for n, w in norms.items()]
    path, extra = str(tmp_path / "model.gguf"), str(tmp_path / "adapter.gguf")
    _write(path, tensors, qwen35__rope__freq_base=1e7, qwen35__rope__dimension_count=16, qwen35__attention__layer_norm_rms_epsilon=1e-5)
    model = loader.load_gguf(path)
    att = model.attention(3)
    assert (att.n_heads, att.n_kv_heads, att.head_dim, att.gated) == (8, 2, 64, True) and att.inv_freq.numel() == 8 and abs(att.eps - 1e-5) < 1e-9
    assert torch.equal(att.q_norm, torch.from_numpy(norms["q"]).to(torch.bfloat16).cuda()) and torch.equal(att.inv_freq, ops.rotary_frequencies(16, 1e7)[0])
    assert model.attention(3, rotary_dim=64, scaling="linear", factor=2.0).inv_freq.numel() == 32
    pairs = {"attn_q": (1024, k), "attn_v": (128, k), "attn_output": (k, 512), "ffn_up": (768, k)}
    r, mats = 6, []
    for n, (no, kk) in pairs.items():
        mats += [(f"blk.3.{n}.weight.lora_a", rng.standard_normal((r, kk)).astype(np.float32) / 20, None), (f"blk.3.{n}.weight.lora_b", rng.standard_normal((no, r)).astype(np.float16), None)]
    half = torch.from_numpy(mats[-1][1]).to(torch.bfloat16)                # one of them as BF16, which the file holds as bytes
    mats[-1] = (mats[-1][0], half.view(torch.uint8).numpy(), 30)
    _write(extra, mats, general__type="adapter", adapter__type="lora", adapter__lora__alpha=12.0)
    with pytest.raises(ValueError, match="add_adapters"):
        loader.load_adapter(extra, model, 0)
    model.add_adapters(2, 8)
    assert loader.load_adapter(extra, model, 1, scale=0.5) == ["layers.3.mlp.gate_up_proj", "layers.3.self_attn.o_proj", "layers.3.self_attn.qkv_proj"]
    x = synth.activations(5, k, device="cuda")
    raw = {n: a if t is None else half.float().numpy() for n, a, t in mats}
    for key, shards in (("layers.3.self_attn.qkv_proj", (("attn_q", 0, 1024), ("attn_k", 1024, 128), ("attn_v", 1152, 128))), ("layers.3.mlp.gate_up_proj", (("ffn_gate", 0, 768), ("ffn_up", 768, 768)))):
        lin = model.linears[key]
        got, base = lin(x, adapters=torch.tensor([1, 0, -1, 1, 1], device="cuda")), lin(x)
        assert torch.equal(got[1:3], base[1:3])                   # an empty slot, no adapter
        for n, at, rows in shards:
            if n not in pairs:
                assert torch.equal(got[:, at:at + rows], base[:, at:at + rows])
                continue
            a, b = torch.from_numpy(raw[f"blk.3.{n}.weight.lora_a"]).to(torch.bfloat16).double().cuda(), torch.from_numpy(raw[f"blk.3.{n}.weight.lora_b"]).to(torch.bfloat16).double().cuda()
            want = base[:, at:at + rows].double() + 12.0 / r * 0.5 * (x.double() @ a.T @ b.T)
            size = base[:, at:at + rows].double().abs() + 12.0 / r * 0.5 * (x.double().abs() @ a.abs().T @ b.abs().T)
            err = ((got[:, at:at + rows].double() - want).abs() - 2.0 ** -8 * want.abs() - 2.0 ** -14 * size)[[0, 3, 4]]      # one rounding; sums of 512 + 8 terms and the inner values' parts
            assert bool((err <= 0).all())
    for bad, why in (([("blk.9.attn_q.weight.lora_a", np.zeros((4, k), np.float32), None), ("blk.9.attn_q.weight.lora_b", np.zeros((1024, 4), np.float32), None)], "no layer"),
                     ([("blk.3.attn_q.weight.lora_a", np.zeros((4, k), np.float32), None)], "half"), ([("blk.3.attn_q.weight", np.zeros((4, k), np.float32), None)], "pair")):
        _write(str(tmp_path / "bad.gguf"), bad, adapter__type="lora")
        with pytest.raises(ValueError, match=why):
            loader.load_adapter(str(tmp_path / "bad.gguf"), model, 1)
    with pytest.raises(ValueError, match="not a low-rank adapter"):
        loader.load_adapter(path, model, 0)
    cache = att.cache(4)
    table = torch.arange(4, device="cuda").view(1, 4).int()
    pos = torch.arange(5, device="cuda")
    y = att(x, pos, cache, cache.slots(table, torch.zeros(5, device="cuda"), pos), table, torch.tensor([5], dtype=torch.int32, device="cuda"), adapters=torch.ones(5, dtype=torch.int64, device="cuda"))
    assert y.shape == (5, k) and bool(y.isfinite().all())


def test_the_traced_forms_give_the_same():
    s = adapters.make(9, 512, (64, 40), 16, 3)
    args = [s[n] for n in ("base", "x", "a", "b", "scales", "ids", "n_outs")]
    assert torch.equal(torch.ops.gq_b200.low_rank_add(*args), adapters.call(s))
    p, more, _ = paged.make([50, 20], [2, 2], 4, 2, 64, 16)
    want = ops.paged_attention(**p)
    assert torch.equal(torch.ops.gq_b200.paged_attention(p["q"], p["k_pages"], p["v_pages"], p["page_table"], p["lens"], None, None, None, None), want)
    inv, _ = ops.rotary_frequencies(64)
    qkv, pos = adapters.bf16(6, 8 * 64, seed=3), torch.arange(6, device="cuda")
    how = (pos, inv, 4, 2, 64, None, None, 1e-6, 1.0, False, False)
    q, k = torch.ops.gq_b200.qk_norm_rope(qkv, *how)
    assert all(torch.equal(a, b) for a, b in zip((q, k), ops.qk_norm_rope(qkv, pos, inv, 4, 2, 64)))
    cache = PagedKVCache(2, 16, 2, 64)
    assert torch.equal(torch.ops.gq_b200.qk_norm_rope_store(qkv, *how, cache.k, cache.v, pos + 3), q)
    assert torch.equal(cache.k.reshape(32, 2, 64)[3:9], k)


def test_a_gradient_is_refused():
    s = adapters.make(2, 256, (16,), 8, 1)
    s["x"].requires_grad_(True)
    with pytest.raises(ops.GqError, match="no backward"):
        adapters.call(s)
    with torch.no_grad():
        adapters.check(adapters.call(s), {**s, "x": s["x"].detach()})


def test_calls_of_nothing():
    s = adapters.make(3, 256, (24, 8), 8, 2)
    none = {**s, "x": s["x"][:0], "base": s["base"][:0], "ids": s["ids"][:0]}
    assert adapters.call(none).shape == (0, 32)
    assert adapters.call({**s, "base": s["base"][:, :0], "b": s["b"][:, :0], "n_outs": [0, 0]}).shape == (3, 0)
    inv, _ = ops.rotary_frequencies(16)
    cache = PagedKVCache(2, 16, 1, 64)
    qkv = adapters.bf16(0, 4 * 64, seed=1)
    at = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.qk_norm_rope(qkv, at, inv, 2, 1, 64)[1].shape == (0, 1, 64)
    assert ops.qk_norm_rope_store(qkv, at, inv, 2, 1, 64, cache.k, cache.v, at).shape == (0, 2, 64)
    table, lens = torch.zeros(0, 4, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(adapters.bf16(0, 2, 64, seed=1), cache.k, cache.v, table, lens).shape == (0, 2, 64)
    q = adapters.bf16(3, 2, 64, seed=2)
    no_keys = ops.paged_attention(q, cache.k, cache.v, torch.zeros(3, 0, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert bool((no_keys == 0).all()) and ops.device_status() == 0
    for pages, width in ((cache.k[:0], 4), (cache.k, 0)):          # keys, but no cache or no table
        got = ops.paged_attention(q, pages, pages, torch.zeros(3, width, dtype=torch.int32, device="cuda"), torch.tensor([0, 5, 0], dtype=torch.int32, device="cuda"))
        assert bool(got[1].isnan().all()) and bool((got[[0, 2]] == 0).all())
        assert ops.device_status() == 2


def test_the_first_call_of_a_process_may_be_captured():
    """In a process of its own: every operator's first call is inside a capture; replayed, it gives what the next, eager one gives."""
    import os
    import subprocess
    import sys

    program = """
import torch
import test_gpu_adapters as adapters, test_gpu_paged as paged
from hyperqwen_rtx4080s32_b200 import ops
few, many = adapters.make(3, 512, (64, 32), 16, 2), adapters.make(200, 512, (64, 32), 16, 2)
p, more, _ = paged.make([300, 40], [1, 1], 8, 2, 128, 16)
inv, _ = ops.rotary_frequencies(64)
qkv, pos = adapters.bf16(6, 8 * 64, seed=3), torch.arange(6, device="cuda")
calls = [lambda: adapters.call(few), lambda: adapters.call(many), lambda: ops.paged_attention(**p), lambda: ops.qk_norm_rope(qkv, pos, inv, 4, 2, 64)[0]]
torch.cuda.synchronize()
for call in calls:
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call())
print("captured")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here), os.environ.get("PYTHONPATH", "")]))
    run = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, env=env, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]


def test_memory_that_is_written_and_read_is_refused():
    s = adapters.make(4, 256, (256,), 8, 1)
    both = torch.zeros(6, 256, dtype=torch.bfloat16, device="cuda")
    for base, out in ((both[:4], both[1:5]), (both[1:5], both[:4])):
        with pytest.raises(ops.GqError, match="base itself"):
            adapters.call({**s, "base": base}, out=out)
    for name in ("x", "b"):
        with pytest.raises(ops.GqError, match="input other than base"):
            adapters.call(s, out=s[name].view(-1)[:1024].view(4, 256))
    p, more, _ = paged.make([20, 30], [1, 1], 4, 2, 64, 16)
    for out in (p["q"], p["v_pages"].transpose(1, 2).view(-1)[:512].view(2, 4, 64)):
        with pytest.raises(ops.GqError, match="shares no memory"):
            ops.paged_attention(**p, out=out)
    cache = PagedKVCache(2, 16, 2, 64)
    inv, _ = ops.rotary_frequencies(64)
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ops.GqError, match="share no memory"):
        ops.qk_norm_rope_store(cache.v.transpose(1, 2).view(-1)[:1024].view(2, 512), pos, inv, 4, 2, 64, cache.k, cache.v, pos)
    with pytest.raises(ops.GqError, match="CUDA"):
        adapters.call({**s, "scales": s["scales"].cpu()})


def test_modes_and_tracers_see_the_calls():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    s = adapters.make(5, 256, (24, 8), 8, 2)
    p, _, _ = paged.make([30, 20], [1, 1], 4, 2, 64, 16)
    inv, _ = ops.rotary_frequencies(64)
    qkv, pos = adapters.bf16(6, 8 * 64, seed=3), torch.arange(6, device="cuda")
    cache = PagedKVCache(2, 16, 2, 64)
    calls = [lambda: adapters.call(s), lambda: adapters.call({**s, "base": s["base"].clone()}, out=torch.empty_like(s["base"])), lambda: ops.paged_attention(**p),
             lambda: ops.paged_attention(**p, out=torch.empty_like(p["q"])), lambda: ops.qk_norm_rope(qkv, pos, inv, 4, 2, 64)[1], lambda: ops.qk_norm_rope_store(qkv, pos, inv, 4, 2, 64, cache.k, cache.v, pos)]
    for call in calls:
        want = call()
        with torch.device("cuda"):
            assert torch.equal(call(), want)
        with torch.autocast("cuda", dtype=torch.bfloat16), torch.inference_mode():
            assert torch.equal(call(), want)
        with Names() as names:
            got = call()
        assert torch.equal(got, want) and any("gq_b200" in n for n in names.seen)
    traced = torch.jit.trace(lambda q: ops.paged_attention(q, *[p[n] for n in ("k_pages", "v_pages", "page_table", "lens")]), (p["q"],), check_trace=False)
    other = p["q"] * 0.5
    assert torch.equal(traced(other), ops.paged_attention(**{**p, "q": other}))
    wrong = [lambda: adapters.call(s, out=torch.empty(2, *s["base"].shape, dtype=torch.bfloat16, device="cuda")), lambda: adapters.call(s, out=torch.empty_like(s["base"]).float()),
             lambda: adapters.call(s, out=torch.empty_like(s["base"], device="cpu")), lambda: adapters.call({**s, "x": s["x"].clone().requires_grad_()}),
             lambda: ops.paged_attention(**{**p, "q": p["q"].clone().requires_grad_()}), lambda: ops.paged_attention(**p, out=torch.empty(2, *p["q"].shape, dtype=torch.bfloat16, device="cuda"))]
    for call in wrong:
        with pytest.raises(ops.GqError):
            call()
        with torch.device("cuda"), Names(), pytest.raises(ops.GqError):
            call()
