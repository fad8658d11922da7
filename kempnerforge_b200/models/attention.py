"""Grouped-query attention with rotary embeddings.

One GEMM produces q, k and v (their weights are adjacent in the block's flat
parameter buffer), one kernel rotates the q and k heads in place of the six
elementwise ops of a naive RoPE, and the attention kernel reads KV head
``h // (n_heads // n_kv_heads)`` directly, so grouped KV heads are never
expanded.  Document masks are evaluated inside the kernel from per-token ids;
no (S, S) mask tensor is built on the native path.

Parity: kempnerforge/model/attention.py:29-280 (parameter names q/k/v/o_proj,
optional per-head q_norm/k_norm applied before RoPE, KV cache for decoding,
``capture_attention_weights`` / ``last_attention_weights`` for inspection,
causal / document / key-padding masks, scale 1/sqrt(head_dim)).
"""

from __future__ import annotations

import torch
from torch import nn

from kempnerforge_b200.models.norm import RMSNorm
from kempnerforge_b200.ops import functional as F
from kempnerforge_b200.ops import ref


class KVCache:
    """Pre-allocated keys/values for incremental decoding, stored (batch, position, kv_head, head_dim)."""

    def __init__(self, batch_size, max_seq_len, n_kv_heads, head_dim, dtype, device) -> None:
        shape = (batch_size, max_seq_len, n_kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.seq_len = 0

    def update(self, k_new: torch.Tensor, v_new: torch.Tensor):
        """Append (batch, new, kv_head, head_dim) entries; returns views over everything cached so far."""
        end = self.seq_len + k_new.shape[1]
        if end > self.k.shape[1]:
            raise ValueError(f"KV cache overflow: {end} > {self.k.shape[1]}")
        self.k[:, self.seq_len : end] = k_new
        self.v[:, self.seq_len : end] = v_new
        self.seq_len = end
        return self.k[:, :end], self.v[:, :end]

    def reset(self) -> None:
        self.seq_len = 0


class SharedPrefixCache:
    """Keys and values of ``width`` continuations of each prompt of a batch: the prompts' own, once, and those of each continuation's
    tokens, (batch, width, position, kv_head, head_dim).  A generation step over it has batch x width rows, the continuations of a
    prompt side by side.

    ``rows`` (batch, width, position) uint8, shared by all layers: in which continuation's cache a position lies.  Beams are exchanged by
    :func:`kempnerforge_b200.ops.beam.reorder` of the rows alone; the keys stay where they are.
    """

    def __init__(self, prefix: KVCache, width: int, max_new: int, rows: torch.Tensor | None = None) -> None:
        n = prefix.seq_len
        self.k, self.v = prefix.k[:, :n], prefix.v[:, :n]
        shape = (self.k.shape[0], width, max_new, *self.k.shape[2:])
        self.own_k = torch.zeros(shape, dtype=self.k.dtype, device=self.k.device)
        self.own_v = torch.zeros(shape, dtype=self.v.dtype, device=self.v.device)
        self.rows, self.width, self.prefix_len, self.seq_len = rows, width, n, n

    @staticmethod
    def new_rows(batch: int, width: int, max_new: int, device) -> torch.Tensor:
        """Every position in its own continuation's cache."""
        if width > 256:
            raise ValueError(f"{width} continuations: their numbers are bytes")
        room = -(-max_new // 16) * 16   # beams on 16 bytes, which a reordering moves in one word
        own = torch.arange(width, device=device, dtype=torch.uint8)[None, :, None]
        return own.expand(batch, width, room).contiguous()[:, :, :max_new]

    def attend(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor) -> torch.Tensor:
        """Append one position (batch x width, 1, kv_head, head_dim) and attend to all: q (batch x width, 1, heads, head_dim)."""
        at, b, w = self.seq_len - self.prefix_len, self.k.shape[0], self.width
        if q.shape[0] != b * w or q.shape[1] != 1 or k_new.shape[:2] != q.shape[:2]:
            raise ValueError(f"one new token for each of {b} x {w} continuations, not {tuple(q.shape[:2])}")
        if at >= self.own_k.shape[2]:
            raise ValueError(f"KV cache overflow: {at + 1} > {self.own_k.shape[2]} new tokens")
        self.own_k[:, :, at] = k_new.reshape(b, w, *k_new.shape[2:])
        self.own_v[:, :, at] = v_new.reshape(b, w, *v_new.shape[2:])
        self.seq_len += 1
        rows = None if self.rows is None else self.rows[:, :, : at + 1]
        out = F.shared_prefix_attention(q.view(b, w, *q.shape[2:]), self.k, self.v, self.own_k[:, :, : at + 1], self.own_v[:, :, : at + 1],
                                        own_rows=rows)
        return out.view(q.shape)


class Attention(nn.Module):
    def __init__(
        self,
        dim: int,
        n_heads: int,
        n_kv_heads: int,
        head_dim: int | None = None,
        qk_norm: bool = False,
        sdpa_backend: str = "auto",
    ) -> None:
        super().__init__()
        self.n_heads = n_heads
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim or dim // n_heads
        self.n_rep = n_heads // n_kv_heads
        self.sdpa_backend = sdpa_backend
        hd = self.head_dim
        self.q_proj = nn.Linear(dim, n_heads * hd, bias=False)
        self.k_proj = nn.Linear(dim, n_kv_heads * hd, bias=False)
        self.v_proj = nn.Linear(dim, n_kv_heads * hd, bias=False)
        self.o_proj = nn.Linear(n_heads * hd, dim, bias=False)
        self.q_norm = RMSNorm(hd) if qk_norm else None
        self.k_norm = RMSNorm(hd) if qk_norm else None
        self.capture_attention_weights = False
        self.last_attention_weights: torch.Tensor | None = None
        self.tp = None  # TPContext when q/k/v are column-sharded and o row-sharded

    def forward(
        self,
        x: torch.Tensor,
        rope_cos: torch.Tensor,
        rope_sin: torch.Tensor,
        kv_cache: KVCache | SharedPrefixCache | None = None,
        doc_ids: torch.Tensor | None = None,
        key_padding_mask: torch.Tensor | None = None,
        qkv: torch.Tensor | None = None,
    ) -> torch.Tensor:
        """``qkv``: the three projections (.., q | k | v) where the caller has them already; ``x`` then gives the shape only."""
        qkv_w = [self.q_proj.weight, self.k_proj.weight, self.v_proj.weight]
        if (qkv is None and x.is_cuda and self.tp is None and self.q_norm is None and kv_cache is None and key_padding_mask is None
                and not self.capture_attention_weights):
            out = F.qkv_attention(x, *qkv_w, rope_cos, rope_sin, doc_ids, self.head_dim)
            if out is not None:
                return F.linear(out, self.o_proj.weight)
        if self.tp is not None:
            qkv = self.tp.column_linear(x, qkv_w)  # gathers the sequence shards (inside the GEMM when it can)
            b, s = qkv.shape[0], qkv.shape[1]
        else:
            b, s, _ = x.shape
        # local head counts follow the weight shapes so a tensor-parallel shard works unchanged
        hd = self.head_dim
        h = self.q_proj.weight.shape[0] // hd
        hkv = self.k_proj.weight.shape[0] // hd
        if qkv is None:
            qkv = F.fused_linear(x, qkv_w)
        qkv = qkv.view(b, s, h + 2 * hkv, hd)
        if self.q_norm is not None:
            qkv = torch.cat(
                [self.q_norm(qkv[:, :, :h]), self.k_norm(qkv[:, :, h : h + hkv]), qkv[:, :, h + hkv :]], dim=2
            )
        qkv = F.rope(qkv, rope_cos, rope_sin, n_rot_heads=h + hkv)
        q, k, v = qkv[:, :, :h], qkv[:, :, h : h + hkv], qkv[:, :, h + hkv :]
        shared = isinstance(kv_cache, SharedPrefixCache)
        if shared and (doc_ids is not None or key_padding_mask is not None or self.capture_attention_weights):
            raise ValueError("a step over a shared prefix takes no masks and keeps no attention weights")
        if kv_cache is not None and not shared:
            k, v = kv_cache.update(k, v)
        causal = kv_cache is None or s > 1
        if shared:
            out = kv_cache.attend(q, k, v)
        elif self.capture_attention_weights:
            out, probs = ref.attention(q, k, v, causal, doc_ids, key_padding_mask, return_weights=True)
            self.last_attention_weights = probs.detach()
        else:
            out = F.attention(q, k, v, causal=causal, doc_ids=doc_ids, key_padding_mask=key_padding_mask)
        if self.tp is not None:
            return self.tp.row_linear(out.reshape(b, s, h * hd), self.o_proj.weight)
        return F.linear(out.reshape(b, s, h * hd), self.o_proj.weight)
