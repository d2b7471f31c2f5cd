"""Decode caches: per Mamba layer a rolling conv window and the SSM state, per attention layer of a hybrid model pages of keys
and values.

Field names and shapes follow the `Mamba2Cache` of transformers 4.46 that the reference imports
(mamba2/mamba2_mixer.py:23) and the layouts its decode kernel uses
(mamba2/mamba2_kernel_inference.py:36-43): `conv_states[layer]` is `[B, conv_dim, K]` (oldest token
first), `ssm_states[layer]` is `[B, H, P, N]`; sizes are per tensor-parallel rank.  The reference's hybrid has no cache
(mamba2hybrid/mamba2hybrid_attn.py:379); the pages are those of `ops.kv_pages`.
"""
from __future__ import annotations

import contextlib
import math
from typing import Optional

import torch

from .. import ops
from ..parallel import state as ps


_PIECE = 64 << 20


def _zeros(count: int, shape, dtype, device):
    """`count` zero tensors of one shape.  Small ones whose sizes are whole 16-byte vectors share allocations and fills of at most
    64 MB (48 fills took 250 us of the host in front of a prompt through 24 layers); larger ones have one each, so that a cache needs
    no more memory in one piece than a layer's state, and a layer's state that is kept holds no more than that.  Each has a version
    counter of its own."""
    size = math.prod(shape) * dtype.itemsize
    each = _PIECE // size if size and size % 16 == 0 else 1
    if each < 2:
        return [torch.zeros(shape, device=device, dtype=dtype) for _ in range(count)]
    return [t.data for first in range(0, count, each)
            for t in torch.zeros((min(each, count - first), *shape), device=device, dtype=dtype).unbind(0)]


class Mamba2Cache:
    def __init__(self, config, batch_size: int, dtype: torch.dtype = torch.float16,
                 device: Optional[torch.device] = None, ssm_dtype: torch.dtype = torch.float32,
                 layer_indices=None):
        tp = ps.get_tensor_model_parallel_size()
        self.dtype = dtype
        self.seqlen_offset = 0
        self.conv_kernel_size = config.conv_kernel
        conv_dim = (config.intermediate_size + 2 * config.n_groups * config.state_size) // tp
        heads = config.num_heads // tp
        layers = range(config.num_hidden_layers) if layer_indices is None else layer_indices
        layers = list(layers)
        self.conv_states = dict(zip(layers, _zeros(len(layers), (batch_size, conv_dim, config.conv_kernel), dtype, device)))
        self.ssm_states = dict(zip(layers, _zeros(len(layers), (batch_size, heads, config.head_dim, config.state_size), ssm_dtype,
                                                  device)))

    def update_conv_state(self, layer_idx: int, new_conv_state: torch.Tensor) -> torch.Tensor:
        self.conv_states[layer_idx].copy_(new_conv_state.to(self.conv_states[layer_idx].dtype))
        return self.conv_states[layer_idx]

    def update_ssm_state(self, layer_idx: int, new_ssm_state: torch.Tensor) -> torch.Tensor:
        self.ssm_states[layer_idx].copy_(new_ssm_state.to(self.ssm_states[layer_idx].dtype))
        return self.ssm_states[layer_idx]

    def reset(self) -> None:
        self.seqlen_offset = 0
        for t in list(self.conv_states.values()) + list(self.ssm_states.values()):
            t.zero_()

    def step_state(self):
        """The tensors that a decoding step changes and the next one reads."""
        return list(self.conv_states.values()) + list(self.ssm_states.values())

    def require_room(self, tokens: int) -> None:
        """Raises where the cache cannot take more tokens; the states of Mamba layers always can."""


class Mamba2HybridCache(Mamba2Cache):
    """Cache of a hybrid model: the Mamba layers' states, and for each attention layer a pool of pages (`pages[layer]`,
    `ops.KVPages`) with room for `max_length` tokens of every sequence.  `block_table` [B, pages per sequence] and `lengths` [B]
    (int32, tokens of each sequence) serve all layers.  `kv_dtype`: bfloat16, float8_e4m3fn or int8 (None: `dtype`).

    A prompt that fails leaves the cache empty.  A step that fails between its layers leaves some of them a token ahead of the others:
    the cache is `torn` then, and takes no token until it is reset."""

    def __init__(self, config, batch_size: int, max_length: int, dtype: torch.dtype = torch.bfloat16,
                 device: Optional[torch.device] = None, ssm_dtype: torch.dtype = torch.float32, kv_dtype: Optional[torch.dtype] = None,
                 page_size: int = 64):
        from .layer_allocation import ATTENTION, MAMBA, allocate_layers
        kinds = allocate_layers(config.num_hidden_layers, config.hybrid_attention_ratio, config.hybrid_mlp_ratio,
                                config.hybrid_override_pattern)
        with torch.inference_mode(False):        # ordinary tensors: a cache may be made in inference mode and used outside
            super().__init__(config, batch_size, dtype, device, ssm_dtype, [i for i, k in enumerate(kinds) if k == MAMBA])
            mult = int(getattr(config, "kv_shared_group_size", 1)) if getattr(config, "qkv_linear", False) else 1
            heads = config.attn_key_value_heads * mult // ps.get_tensor_model_parallel_size()
            per = -(-max_length // page_size)
            self.max_length = max_length
            self.pages = {i: ops.kv_pages(batch_size * per, heads, page_size, config.attn_head_dim, kv_dtype or dtype, device)
                          for i, k in enumerate(kinds) if k == ATTENTION}
            self.block_table = torch.arange(batch_size * per, dtype=torch.int32, device=device).view(batch_size, per)
            self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self._tables = {}
        self.torn = False

    def rotary_tables(self, dim: int, theta: float):
        """cos / sin of every position that the cache has room for."""
        if self.lengths.is_cuda:                 # kept there
            return ops.rotary_tables(self.max_length, dim, theta, device=self.lengths.device)
        if (dim, theta) not in self._tables:
            self._tables[dim, theta] = ops.rotary_tables(self.max_length, dim, theta, device=self.lengths.device)
        return self._tables[dim, theta]

    def require_room(self, tokens: int) -> None:
        if self.torn:
            raise RuntimeError("a step over this cache failed between its layers; reset() it")
        self._require_room(tokens)

    def _require_room(self, tokens: int) -> None:
        if self.seqlen_offset + tokens > self.max_length:
            raise ValueError(f"the cache has room for {self.max_length} tokens, holds {self.seqlen_offset} and was given {tokens} more")

    def require_batch(self, batch: int) -> None:
        if batch != self.lengths.shape[0]:
            raise ValueError(f"the cache holds {self.lengths.shape[0]} sequences and was given {batch}")

    def begin(self, tokens: int) -> None:
        """Counts a prompt's tokens in an empty cache (whatever a call that failed has left)."""
        self._require_room(tokens)
        self.torn = False
        self.lengths.fill_(tokens)

    def take(self, tokens: int) -> None:
        """Counts new tokens of every sequence; the attention layers put them behind the others."""
        self.require_room(tokens)
        self.lengths.add_(tokens)

    @contextlib.contextmanager
    def prompt(self, tokens: int):
        """Around the layers that a prompt runs through."""
        self.begin(tokens)
        try:
            yield
        except BaseException:
            self.reset()
            raise
        self.seqlen_offset += tokens

    @contextlib.contextmanager
    def token(self):
        """Around the layers that one token of every sequence runs through."""
        self.take(1)
        self.torn = True
        yield
        self.torn = False
        self.seqlen_offset += 1

    def keys_values(self, layer_idx: int, dtype: torch.dtype = torch.bfloat16):
        """Cached keys and values of an attention layer as the values they stand for, [B, tokens, kv heads, head_dim] each."""
        return ops.kv_cache_read(self.pages[layer_idx], self.block_table, self.lengths, self.seqlen_offset, dtype)

    def step_state(self):
        return super().step_state() + [self.lengths]

    def reset(self) -> None:
        super().reset()
        self.lengths.zero_()
        self.torn = False
