"""Causal grouped-query self-attention block of the hybrid model.

Parameters `q_proj/k_proj/v_proj` (column parallel) and `o_proj` (row parallel), no biases, no
dropout, per-rank heads = attn_num_heads/TP and kv heads = attn_key_value_heads/TP
(mamba2hybrid/mamba2hybrid_attn.py:305-362,491-514).  The three projections share one sequence
all-gather, K/V heads are never replicated in memory (the kernel indexes kv head = q head // ratio,
where the reference materialises `repeat_kv`, mamba2hybrid_attn.py:440-447), and rotary embedding (its own
kernel, forward and backward, with cached tables) is an option that is off by default as in the reference
hybrid (mamba2hybrid_attn.py:500-503).  With `qk_norm` queries and keys are normed per head and rotated in one pass.
A prompt leaves its keys and values in the pages of a `Mamba2HybridCache`; `step` decodes one token over them.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import ops
from ..parallel import mappings as mp
from ..parallel import state as ps
from ..parallel.layers import ColumnParallelLinear, GQAQKVColumnParallelLinear, RowParallelLinear, normal_init


class HeadRMSNorm(nn.Module):
    """Weight of an RMS norm over the channels of a head, shared by the heads; the attention applies it.  Each tensor-parallel rank
    sees its own heads, so the gradient is summed over the group as that of a norm under sequence parallelism is."""

    def __init__(self, head_dim: int, dtype=torch.float32, device=None):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(head_dim, dtype=dtype, device=device))
        if ps.get_tensor_model_parallel_size() > 1:
            self.weight.sequence_parallel_enabled = True


class Mamba2HybridAttention(nn.Module):
    def __init__(self, config, layer_idx: int, device=None):
        super().__init__()
        tp = ps.get_tensor_model_parallel_size()
        self.layer_idx = layer_idx
        self.hidden_size = config.hidden_size
        self.total_heads = config.attn_num_heads
        self.total_kv_heads = config.attn_key_value_heads
        self.head_dim = config.attn_head_dim
        self.qkv_linear = bool(getattr(config, "qkv_linear", False))
        kv_mult = int(getattr(config, "kv_shared_group_size", 1)) if self.qkv_linear else 1
        if self.total_heads % tp or (self.total_kv_heads * kv_mult) % tp:
            raise ValueError("attention heads and kv heads (times kv_shared_group_size) must be divisible by the TP size")
        self.num_heads = self.total_heads // tp
        self.num_kv_heads = self.total_kv_heads * kv_mult // tp
        self.sequence_parallel_enabled = config.sequence_parallel_enabled and tp > 1
        self.rotary_emb_dim = getattr(config, "rotary_emb_dim", None)
        self.rope_theta = getattr(config, "rope_theta", 10000.0)
        dtype = config.dtype or torch.float32
        self.norm_eps = config.layer_norm_epsilon
        qk_norm = bool(getattr(config, "qk_norm", False))
        self.q_norm = HeadRMSNorm(self.head_dim, dtype, device) if qk_norm else None
        self.k_norm = HeadRMSNorm(self.head_dim, dtype, device) if qk_norm else None
        init = normal_init(config.initializer_range)
        kw = dict(bias=False, init_method=init, dtype=dtype, device=device,
                  sequence_parallel_enabled=config.sequence_parallel_enabled)
        if self.qkv_linear:
            # one layer for q, k, v with optional KV-head replication (mamba2hybrid_attn.py:291-303 of the reference)
            self.qkv_proj = GQAQKVColumnParallelLinear(
                self.hidden_size, [self.total_heads * self.head_dim, self.total_kv_heads * self.head_dim],
                kv_size_multiplier=kv_mult, fuse_qkv=bool(getattr(config, "fuse_qkv", False)), head_dim=self.head_dim, **kw)
        else:
            self.q_proj = ColumnParallelLinear(self.hidden_size, self.total_heads * self.head_dim, **kw)
            self.k_proj = ColumnParallelLinear(self.hidden_size, self.total_kv_heads * self.head_dim, **kw)
            self.v_proj = ColumnParallelLinear(self.hidden_size, self.total_kv_heads * self.head_dim, **kw)
        self.o_proj = RowParallelLinear(self.total_heads * self.head_dim, self.hidden_size, bias=False,
                                        init_method=init, dtype=dtype, device=device,
                                        sequence_parallel_enabled=config.sequence_parallel_enabled)

    def _queries_keys_values(self, hidden_states):
        """[B, L, heads, head_dim] each, of the whole sequence."""
        qkv = None
        if self.qkv_linear:
            qkv = self.qkv_proj(hidden_states)
        elif self.sequence_parallel_enabled:
            from ..parallel import fused
            if fused.enabled_for(hidden_states):
                qkv = fused.all_gather_multi_linear(
                    hidden_states, (self.q_proj.weight, self.k_proj.weight, self.v_proj.weight))
            if qkv is None:
                x = mp.gather_from_sequence_parallel_region(hidden_states, True)
        else:
            x = mp.copy_to_tensor_parallel_region(hidden_states)
        if qkv is None:
            qkv = (ops.linear(x, self.q_proj.weight), ops.linear(x, self.k_proj.weight),
                   ops.linear(x, self.v_proj.weight))
        B, L = qkv[0].shape[0], qkv[0].shape[1]
        q = qkv[0].view(B, L, self.num_heads, self.head_dim)
        k = qkv[1].view(B, L, self.num_kv_heads, self.head_dim)
        v = qkv[2].view(B, L, self.num_kv_heads, self.head_dim)
        return q, k, v

    def forward(self, hidden_states: torch.Tensor, cache_params=None) -> torch.Tensor:
        """Whole sequences.  With `cache_params` (a `Mamba2HybridCache` that has counted these tokens) their keys and values go
        into the layer's pages, ready for `step`."""
        q, k, v = self._queries_keys_values(hidden_states)
        B, L = q.shape[:2]
        cos = sin = None
        if self.rotary_emb_dim is not None:
            cos, sin = ops.rotary_tables(L, self.rotary_emb_dim, self.rope_theta, device=q.device)
        if self.q_norm is not None:
            q, k = ops.qk_norm_rotary(q, k, self.q_norm.weight, self.k_norm.weight, self.norm_eps, cos, sin)
        elif cos is not None:
            q = ops.apply_rotary(q, cos, sin)
            k = ops.apply_rotary(k, cos, sin)
        if cache_params is not None:
            ops.kv_cache_write(k, v, cache_params.pages[self.layer_idx], cache_params.block_table, cache_params.lengths)
        o = ops.attention(q, k, v, causal=True)
        return self.o_proj(o.reshape(B, L, self.num_heads * self.head_dim))

    @torch.no_grad()
    def step(self, hidden_states: torch.Tensor, cache_params) -> torch.Tensor:
        """Single-token decode over the cached keys and values; hidden_states [B, 1, D].  Norm, rotation and the write into the
        pages are one kernel, the attention another."""
        assert hidden_states.shape[1] == 1, "step() takes one token at a time"
        if self.sequence_parallel_enabled:
            raise RuntimeError("decode runs without sequence parallelism; build the model with it disabled")
        q, k, v = self._queries_keys_values(hidden_states)
        pages, table, lengths = cache_params.pages[self.layer_idx], cache_params.block_table, cache_params.lengths
        cos = sin = None
        if self.rotary_emb_dim is not None:
            cos, sin = cache_params.rotary_tables(self.rotary_emb_dim, self.rope_theta)
        if self.q_norm is None and cos is None:
            ops.kv_cache_write(k, v, pages, table, lengths)
        else:
            weights = (None, None) if self.q_norm is None else (self.q_norm.weight, self.k_norm.weight)
            q = ops.kv_cache_write(k, v, pages, table, lengths, q=q, q_weight=weights[0], k_weight=weights[1], eps=self.norm_eps,
                                   cos=cos, sin=sin)
        o = ops.paged_attention(q, pages, table, lengths)
        return self.o_proj(o.reshape(o.shape[0], 1, self.num_heads * self.head_dim))
