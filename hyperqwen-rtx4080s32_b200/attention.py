"""The attention half of a decoder block between its quantized layers: qkv_proj, norm and rotation of the heads with the store into a
paged cache, attention over the cache, o_proj.

The reference leaves these steps to vLLM around its linear method.  Outside vLLM a file loaded by loader.load_gguf has
the layers and the head norms' weights; LoadedModel.attention puts them together as a GGUFAttention.  It serves decode and verification
(a few new tokens of each sequence) and chunks of prompts alike, is safe to capture in a CUDA graph, and takes the
same ids of low-rank adapters as the layers do.
"""
from __future__ import annotations

import torch

from . import ops
from ._lib import GqError
from .linear import GGUFLinear


class PagedKVCache:
    """The keys and values of one attention layer: `k` and `v`, bf16 [n_pages, page_size, n_kv_heads, head_dim].  The rows of a head stand together
    within a page, so that a head's part of a page is one run of memory; any other strides serve the ops as well."""

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device="cuda"):
        if n_pages < 1 or page_size < 1:
            raise GqError("a cache has one page of one row or more")
        self.page_size = page_size
        memory = torch.zeros((2, n_pages, n_kv_heads, page_size, head_dim), dtype=torch.bfloat16, device=device)
        self.k, self.v = memory[0].transpose(1, 2), memory[1].transpose(1, 2)

    def slots(self, page_table: torch.Tensor, sequences: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """The slots (int64) of tokens at `positions` of `sequences`, rows of page_table; a negative position has none (-1).  Where the table has no page for a token, or
        one outside the cache, the slot is beyond the cache: the store leaves it out and reports it (device_status 2)."""
        at, seq = positions.clamp(min=0).long(), sequences.long()
        page, (n_seqs, width), n_pages = at // self.page_size, page_table.shape, self.k.shape[0]
        beyond = n_pages * self.page_size
        if page_table.numel() == 0:
            return torch.where(positions < 0, -1, beyond).expand(torch.broadcast_shapes(positions.shape, sequences.shape))
        there = (page < width) & (seq >= 0) & (seq < n_seqs)
        pages = page_table[seq.clamp(0, n_seqs - 1), page.clamp(max=width - 1)].long()       # an index outside the table would end the process's context
        slots = torch.where(there & (pages >= 0) & (pages < n_pages), pages * self.page_size + at % self.page_size, beyond)
        return torch.where(positions < 0, -1, slots)


class GGUFAttention(torch.nn.Module):
    """`qkv` and `o` are the merged projection (shards "q", "k", "v") and the output projection; where the q shard has twice the heads' rows, each
    head is followed by an output gate.  head_dim is 64, 128 or 256.  q_norm, k_norm: bf16 [head_dim] or None.  inv_freq, amplitude: ops.rotary_frequencies."""

    def __init__(self, qkv: GGUFLinear, o: GGUFLinear, head_dim: int, inv_freq: torch.Tensor, *, amplitude: float = 1.0, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False):
        super().__init__()
        if len(qkv.output_partition_sizes) != 3:
            raise GqError("qkv has the shards q, k and v")
        if head_dim not in ops.ATTENTION_HEAD_DIMS:            # paged_attention would refuse it, behind the store into the cache
            raise GqError(f"attention takes heads of {ops.ATTENTION_HEAD_DIMS}, got {head_dim}")
        rows_q, rows_k, rows_v = qkv.output_partition_sizes
        if o.input_size % head_dim or not rows_k or rows_k % head_dim or rows_k != rows_v or o.input_size % rows_k or rows_q not in (o.input_size, 2 * o.input_size):
            raise GqError(f"heads of {head_dim} do not fit q / k / v rows of {rows_q} / {rows_k} / {rows_v} and an output projection of {o.input_size} columns")
        self.qkv, self.o = qkv, o
        self.head_dim, self.n_heads, self.n_kv_heads = head_dim, o.input_size // head_dim, rows_k // head_dim
        self.gated = rows_q == 2 * o.input_size
        self.inv_freq, self.amplitude, self.q_norm, self.k_norm, self.eps, self.interleaved = inv_freq, amplitude, q_norm, k_norm, eps, interleaved

    def cache(self, n_pages: int, page_size: int = 16) -> PagedKVCache:
        return PagedKVCache(n_pages, page_size, self.n_kv_heads, self.head_dim, self.inv_freq.device)

    def forward(self, x: torch.Tensor, positions: torch.Tensor, cache: PagedKVCache, slots: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, *,
                q_starts: torch.Tensor | None = None, pre=None, adapters: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 [T, hidden] of the newest tokens of len(lens) sequences -> [T, hidden].  positions and slots [T] place each token in its sequence and in
        the cache; lens counts a sequence's keys with the new ones; q_starts as in ops.paged_attention.  pre: the op in front of qkv_proj
        (ops.PreAddRMSNorm); adapters: ids of the rows' low-rank adapters, for qkv_proj and o_proj."""
        d = self.head_dim
        qkv = self.qkv(x, pre=pre, adapters=adapters)
        q = ops.qk_norm_rope_store(qkv, positions, self.inv_freq, self.n_heads, self.n_kv_heads, d, cache.k, cache.v, slots, q_norm=self.q_norm, k_norm=self.k_norm,
                                   eps=self.eps, amplitude=self.amplitude, interleaved=self.interleaved, gated=self.gated)
        gate = qkv[:, :2 * self.n_heads * d].unflatten(1, (self.n_heads, 2 * d))[..., d:] if self.gated else None
        out = ops.paged_attention(q, cache.k, cache.v, page_table, lens, q_starts=q_starts, gate=gate)
        return self.o(out.flatten(1), adapters=adapters)
