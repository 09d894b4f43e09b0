"""GGUF file -> the layers of the quantized-linear path.

What the plugin's loader and tensor-name adapter do for `MODEL=*.gguf` (vllm_gguf_plugin/loader.py and
vllm_gguf_plugin/weights_adapter/qwen3_5.py, un-vendored; the reference checks them in
gguf-plugin/test_gguf_rco_cpu.py:84-128 against the tensor list gguf-plugin/iq3s-tensor-names.json of the checkpoint
it serves), narrowed to this path: read the file's tensor table, give every tensor its Hugging Face module name, and
hand the quantized 2-D weights to GGUFLinearMethod's weight loaders — q / k / v and gate / up as the shards of the
merged layers vLLM builds (shard ids "q", "k", "v" and 0, 1) —, which repack them tile-major on the device.  Norms,
convolution and state-space tensors, the vision tower and the projector are not linear-method weights: they are
reported with their names and left to the engine (the head norms of an attention block go into LoadedModel.attention).

The file is read with the `gguf` package (the reference pins gguf==0.17.1, gguf-plugin/requirements.txt:1); tensor data
stay memory-mapped until they are copied to the device, one tensor at a time.
"""
from __future__ import annotations

import re
from dataclasses import dataclass, field
from typing import Iterator

import numpy as np
import torch

from . import formats as F
from .linear import GGUFLinear

# GGUF tensor suffix inside "blk.N." -> (HF module, merged vLLM layer or None, shard id in it)
_BLOCK_LINEAR = {
    "attn_q": ("self_attn.q_proj", "self_attn.qkv_proj", "q"),
    "attn_k": ("self_attn.k_proj", "self_attn.qkv_proj", "k"),
    "attn_v": ("self_attn.v_proj", "self_attn.qkv_proj", "v"),
    "attn_output": ("self_attn.o_proj", None, None),
    "attn_qkv": ("linear_attn.in_proj_qkv", None, None),
    "attn_gate": ("linear_attn.in_proj_z", None, None),
    "ssm_out": ("linear_attn.out_proj", None, None),
    "ffn_gate": ("mlp.gate_proj", "mlp.gate_up_proj", 0),
    "ffn_up": ("mlp.up_proj", "mlp.gate_up_proj", 1),
    "ffn_down": ("mlp.down_proj", None, None),
}
# tensors of a block that are not weights of a linear method
_BLOCK_OTHER = {
    "attn_norm.weight": "input_layernorm.weight", "post_attention_norm.weight": "post_attention_layernorm.weight",
    "attn_q_norm.weight": "self_attn.q_norm.weight", "attn_k_norm.weight": "self_attn.k_norm.weight",
    "ssm_alpha.weight": "linear_attn.in_proj_a.weight", "ssm_beta.weight": "linear_attn.in_proj_b.weight",
    "ssm_conv1d.weight": "linear_attn.conv1d.weight", "ssm_norm.weight": "linear_attn.norm.weight",
    "ssm_dt.bias": "linear_attn.dt_bias", "ssm_a": "linear_attn.A_log",
}
_TOP = {"token_embd.weight": "model.language_model.embed_tokens.weight", "output_norm.weight": "model.language_model.norm.weight",
        "output.weight": "lm_head.weight"}
_GGML_NAMES = {2: "Q4_0", 6: "Q5_0", 8: "Q8_0", 10: "Q2_K", 11: "Q3_K", 12: "Q4_K", 13: "Q5_K", 14: "Q6_K", 16: "IQ2_XXS", 17: "IQ2_XS",
               18: "IQ3_XXS", 19: "IQ1_S", 20: "IQ4_NL", 21: "IQ3_S", 22: "IQ2_S", 23: "IQ4_XS", 29: "IQ1_M", 0: "F32", 1: "F16", 30: "BF16"}


@dataclass(frozen=True)
class MappedName:
    hf_name: str                 # e.g. model.language_model.layers.3.self_attn.q_proj.weight
    layer: int | None            # decoder block, None for top-level tensors
    module: str | None           # HF module inside the block (no ".weight"), None if not a linear weight of a block
    merged: str | None           # the merged vLLM layer this weight is a shard of (qkv_proj, gate_up_proj), if any
    shard_id: object = None      # "q" / "k" / "v" or 0 / 1 inside the merged layer


def map_tensor_name(name: str) -> MappedName | None:
    """GGUF tensor name of the text model -> its Hugging Face name and where it goes; None for names this adapter does not
    know (the vision tower `v.*` and the projector `mm.*` belong to another adapter)."""
    if name in _TOP:
        return MappedName(_TOP[name], None, None, None)
    m = re.fullmatch(r"blk\.(\d+)\.(.+)", name)
    if not m:
        return None
    layer, rest = int(m.group(1)), m.group(2)
    prefix = f"model.language_model.layers.{layer}."
    if rest in _BLOCK_OTHER:
        return MappedName(prefix + _BLOCK_OTHER[rest], layer, None, None)
    if rest.endswith(".weight") and rest[:-7] in _BLOCK_LINEAR:
        module, merged, sid = _BLOCK_LINEAR[rest[:-7]]
        return MappedName(prefix + module + ".weight", layer, module, merged, sid)
    return None


@dataclass
class GGUFTensor:
    name: str
    ggml_type: int
    shape: tuple[int, ...]       # logical shape, outermost first: (n_out, K) for a 2-D weight
    data: np.ndarray             # quantized: uint8 [n_out, row_bytes]; otherwise the values

    @property
    def type_name(self) -> str:
        return _GGML_NAMES.get(self.ggml_type, str(self.ggml_type))


def read_gguf(path: str) -> Iterator[GGUFTensor]:
    """The file's tensors in file order (data memory-mapped by the gguf package)."""
    from gguf import GGUFReader

    yield from _tensors(GGUFReader(path))


def _tensors(reader) -> Iterator[GGUFTensor]:
    for t in reader.tensors:
        shape = tuple(int(d) for d in reversed(t.shape))          # GGUF lists the innermost dimension first
        yield GGUFTensor(str(t.name), int(t.tensor_type), shape, t.data)


@dataclass
class LoadedModel:
    linears: dict[str, GGUFLinear] = field(default_factory=dict)   # "layers.3.self_attn.qkv_proj" / "lm_head" -> layer, finalized
    embedding: GGUFTensor | None = None                            # token_embd.weight, left raw (its rows are gathered)
    other: dict[str, GGUFTensor] = field(default_factory=dict)     # HF name -> norms etc., for the engine
    unmapped: list[str] = field(default_factory=list)              # names this adapter does not know
    unsupported: dict[str, str] = field(default_factory=dict)      # linear weights in a GGML type the kernels do not decode
    meta: dict[str, object] = field(default_factory=dict)          # the file's numbers and texts, keys without the architecture: "rope.freq_base"

    def add_adapters(self, n_adapters: int, rank: int) -> None:
        """A bank of low-rank adapters beside every linear layer of the decoder blocks (load_adapter fills them)."""
        for name, lin in self.linears.items():
            if name.startswith("layers."):
                lin.quant_method.add_adapters(lin, n_adapters, rank)

    def _beyond_the_block(self, own_scaling: bool) -> list[str]:
        """What the file says about its attention that GGUFAttention does not do: it would be left out without a word."""
        meta = self.meta
        neutral = {"attention.sliding_window": 0, "attention.scale": 0.0, "attn_logit_softcapping": 0.0, "attention.max_alibi_bias": 0.0, "attention.clamp_kqv": 0.0, "attention.causal": True}
        found = [k for k, v in neutral.items() if meta.get(k, v) != v]
        if not own_scaling:
            neutral = {"attn_factor": 1.0, "yarn_attn_factor": 1.0, "yarn_ext_factor": 1.0, "yarn_log_multiplier": 0.0, "alpha": 0.0}
            found += [f"rope.scaling.{k}" for k, v in neutral.items() if meta.get(f"rope.scaling.{k}", v) != v]
            found += [n for n in self.unmapped if re.search(r"(^|\.)rope_(freqs|factors_long|factors_short)\.weight$", n)]
            if "rope.scaling.type" not in meta and meta.get("rope.scaling.factor", 1.0) not in (0.0, 1.0):
                found.append("rope.scaling.factor without a type")
        return found

    def attention(self, layer: int, *, head_dim: int | None = None, interleaved: bool = False, **rotary):
        """The attention half of a block (attention.GGUFAttention) from its qkv_proj, o_proj and head norms.  What the file says about heads, rotation and eps is
        taken from it; `head_dim` and the arguments of ops.rotary_frequencies (rotary_dim, base, scaling, factor, original_context, beta_fast, beta_slow) go before.  A token has
        one position (text); `interleaved` where the architecture turns neighbours, which the file does not say.  A file that says what this attention does not do (a sliding
        window, rotation factors of its own, ...) raises ValueError; with `scaling` given, what it says about scaling is not looked at."""
        from . import ops
        from .attention import GGUFAttention

        def norm(which):
            t = self.other.get(f"model.language_model.layers.{layer}.self_attn.{which}_norm.weight")
            return None if t is None else _values(t).to(device=device, dtype=torch.bfloat16)

        qkv, o, meta = self.linears[f"layers.{layer}.self_attn.qkv_proj"], self.linears[f"layers.{layer}.self_attn.o_proj"], self.meta
        device = next(iter(qkv.gguf_groups.values()))[0].device
        q_norm, k_norm = norm("q"), norm("k")
        head_dim = head_dim or (q_norm.numel() if q_norm is not None else None) or meta.get("attention.key_length")
        if not head_dim:
            raise ValueError("neither the file nor the call says how wide a head is")
        known = {"rotary_dim": meta.get("rope.dimension_count", head_dim), "base": meta.get("rope.freq_base", 10000.0), "scaling": meta.get("rope.scaling.type"),
                 "factor": meta.get("rope.scaling.factor", 1.0), "original_context": meta.get("rope.scaling.original_context_length"),
                 "beta_fast": meta.get("rope.scaling.yarn_beta_fast", 32.0), "beta_slow": meta.get("rope.scaling.yarn_beta_slow", 1.0)}
        unknown = self._beyond_the_block("scaling" in rotary)
        if unknown:
            raise ValueError(f"layer {layer}: the file says what this attention does not do ({', '.join(unknown)}); attention.GGUFAttention takes frequencies and an amplitude of your own")
        inv_freq, amplitude = ops.rotary_frequencies(**{**known, **rotary}, device=device)
        return GGUFAttention(qkv, o, int(head_dim), inv_freq, amplitude=amplitude, q_norm=q_norm, k_norm=k_norm, eps=float(meta.get("attention.layer_norm_rms_epsilon", 1e-6)),
                             interleaved=interleaved)


def load_gguf(path: str, device="cuda", strict: bool = True) -> LoadedModel:
    """Read a GGUF file and build the path's layers: one GGUFLinear per linear module of the text model, with q / k / v
    and gate / up fused as vLLM fuses them; every weight goes through GGUFLinearMethod's weight loaders and is repacked
    tile-major on `device`.  With strict, a linear weight in a type the kernels do not decode raises; otherwise it is listed
    in `unsupported` and its module is left out."""
    from gguf import GGUFReader

    reader = GGUFReader(path)
    out = LoadedModel(meta=_metadata(reader))
    pending: dict[str, list[tuple[object, GGUFTensor]]] = {}
    order = {"q": 0, "k": 1, "v": 2, 0: 0, 1: 1, None: 0}
    for t in _tensors(reader):
        mapped = map_tensor_name(t.name)
        if mapped is None:
            out.unmapped.append(t.name)
            continue
        if t.name == "token_embd.weight":
            out.embedding = t
            continue
        is_linear = mapped.module is not None or t.name == "output.weight"
        if not is_linear or len(t.shape) != 2 or t.ggml_type in (0, 1, 30):
            out.other[mapped.hf_name] = t
            continue
        if t.ggml_type not in F.SUPPORTED_TYPES:
            if strict:
                raise ValueError(f"{t.name}: GGML type {t.type_name} is not a type the kernels decode")
            out.unsupported[t.name] = t.type_name
            continue
        key = "lm_head" if mapped.layer is None else f"layers.{mapped.layer}.{mapped.merged or mapped.module}"
        pending.setdefault(key, []).append((mapped.shard_id, t))
    for key, shards in pending.items():
        shards.sort(key=lambda s: order[s[0]])
        k = shards[0][1].shape[1]
        if any(t.shape[1] != k for _, t in shards):
            raise ValueError(f"{key}: shards disagree on K")
        lin = GGUFLinear(k, [t.shape[0] for _, t in shards])
        for sid, t in shards:
            want = F.raw_row_bytes(t.ggml_type, k)
            raw = torch.from_numpy(np.array(t.data, copy=True)).reshape(t.shape[0], -1)
            if raw.shape[1] != want:
                raise ValueError(f"{t.name}: {raw.shape[1]} bytes per row, {want} expected for {t.type_name} at K={k}")
            lin.load_shard(raw.to(device), t.ggml_type, sid)
        out.linears[key] = lin.finalize()
    return out


def _values(t: GGUFTensor) -> torch.Tensor:
    """A copy of an F32, F16 or BF16 tensor (the reader gives the last as bytes)."""
    data = torch.from_numpy(np.array(t.data, copy=True))
    return (data.view(torch.bfloat16) if t.ggml_type == 30 else data).reshape(t.shape)


def _metadata(reader) -> dict[str, object]:
    """The file's single numbers and texts; "qwen35.rope.freq_base" is listed as "rope.freq_base" too."""
    out: dict[str, object] = {}
    for name, f in reader.fields.items():
        if len(f.types) == 1 and len(f.data) == 1:
            v = f.contents()
            if isinstance(v, (int, float, str, bool)):
                out[name] = v
    arch = str(out.get("general.architecture", ""))
    return {**out, **{k[len(arch) + 1:]: v for k, v in out.items() if arch and k.startswith(arch + ".")}}


def load_adapter(path: str, model: LoadedModel, slot: int, scale: float = 1.0) -> list[str]:
    """Reads a GGUF adapter file (general.type "adapter", adapter.type "lora": a pair X.lora_a [r, K], X.lora_b [n_out, r] for every adapted weight X, and
    adapter.lora.alpha) into `slot` of the banks that model.add_adapters made, which is emptied first; its products count alpha / r * scale.
    Returns the layers that have it.  Nothing is changed where the file does not fit: a weight that is no linear layer of the model raises ValueError, a slot or
    matrices that are not a bank's GqError."""
    from gguf import GGUFReader

    reader = GGUFReader(path)
    meta = _metadata(reader)
    if meta.get("adapter.type") != "lora":
        raise ValueError(f"{path} is not a low-rank adapter")
    parts: dict[str, dict[str, torch.Tensor]] = {}
    for t in _tensors(reader):
        name, _, which = t.name.rpartition(".lora_")
        if which not in ("a", "b") or t.ggml_type not in (0, 1, 30):
            raise ValueError(f"{t.name}: not one of a pair of matrices in F32, F16 or BF16")
        parts.setdefault(name, {})[which] = _values(t)
    found = []
    for name, pair in parts.items():
        mapped = map_tensor_name(name)
        key = None if mapped is None or mapped.layer is None or mapped.module is None else f"layers.{mapped.layer}.{mapped.merged or mapped.module}"
        lin = model.linears.get(key) if key else None
        if lin is None or len(pair) != 2:
            raise ValueError(f"{name}: no layer of the model, or half of an adapter")
        bank = getattr(lin, "gguf_adapters", None)
        if bank is None or pair["a"].shape[0] > bank.rank:
            raise ValueError(f"{name}: model.add_adapters(rank >= {pair['a'].shape[0]}) comes first")
        bank.check(slot, pair["a"], pair["b"], mapped.shard_id)
        found.append((key, bank, pair, mapped.shard_id))
    banks = [lin.gguf_adapters for lin in model.linears.values() if getattr(lin, "gguf_adapters", None) is not None]
    for bank in banks:
        bank.check_slot(slot)
    for bank in banks:
        bank.clear(slot)
    alpha = float(meta.get("adapter.lora.alpha", 0.0))
    for _, bank, pair, shard_id in found:
        r = pair["a"].shape[0]
        bank.load(slot, pair["a"], pair["b"], scale * (alpha / r if alpha else 1.0), shard_id)
    return sorted({key for key, *_ in found})


def embedding_lookup(raw: torch.Tensor, wtype: int, ids: torch.Tensor, dtype=torch.bfloat16) -> torch.Tensor:
    """Rows `ids` of a quantized embedding table raw uint8 [vocab, row_bytes] (kept raw, as the plugin keeps it:
    gguf-tiles-all-types.patch:80-89) dequantised to [*ids.shape, K]: one launch gathers the rows' bytes and decodes
    them with the decoders that serve the weights — bit-identical to gguf.quants.dequantize of those rows.

    An id outside the table: in host memory it raises IndexError.  On the device nothing can be raised without waiting for it; its
    row is not read, its output is NaN, and ops.device_status (GGUFLinearMethod.check_status, which an engine calls between steps)
    reports 2."""
    from . import ops

    if int(wtype) not in F.SUPPORTED_TYPES:
        raise ValueError(f"GGML type {wtype} is not a type the kernels decode")
    return ops.dequantize_rows(raw, int(wtype), ids, dtype=dtype)
