"""Paged key-value cache: the tensors of one attention layer and what every operation on them checks.

A page holds `page_size` tokens of every key/value head, a head's tokens one behind the other: `k` and `v` are
[pages, kv_heads, page_size, head_dim].  A sequence's token at position p is in slot p % page_size of the page that
`block_table[sequence, p // page_size]` names; sequences share the pool and their pages are in any order.  The head comes before
the token so that the attention kernel reads a head's page as one piece of page_size * head_dim values.

Values are bfloat16, or 8-bit (float8_e4m3fn, int8) with one fp32 scale per token and head in `k_scale` / `v_scale`
[pages, kv_heads, page_size]; a stored value stands for value * scale.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

QUANT_MAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
# Rows whose largest magnitude is below this are stored as zeros with scale 0: the reciprocal of their scale is no fp32 number.
QUANT_TINY = 2.0 ** -100
HEAD_DIMS = (64, 128, 256)


class KVPages(NamedTuple):
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def kv_pages(num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype=torch.bfloat16, device=None) -> KVPages:
    """Zeroed pages of one layer; `dtype` bfloat16, float8_e4m3fn or int8 (CPU: any floating type as well)."""
    shape = (num_pages, kv_heads, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype not in QUANT_MAX:
        return KVPages(k, v)
    return KVPages(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


def check_pages(pages, block_table, lengths, batch: int, counts=None) -> None:
    """What holds for every operation on a cache; raises TypeError or ValueError."""
    k, v, ks, vs = pages
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v pages are [pages, kv_heads, page_size, head_dim] of one shape and type, got "
                         f"{tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    page = k.shape[2]
    if page < 16 or page & (page - 1):
        raise ValueError(f"a page holds a power of two of at least 16 tokens, got {page}")
    if (ks is None) != (vs is None) or (ks is not None) != (k.dtype in QUANT_MAX):
        raise ValueError("8-bit pages come with scales for keys and values, other pages with none")
    for s in (ks, vs):
        if s is not None and (s.shape != k.shape[:3] or s.dtype != torch.float32):
            raise ValueError(f"scales are fp32 of shape {tuple(k.shape[:3])}, got {s.dtype} {tuple(s.shape)}")
    if any(t is not None and not t.is_contiguous() for t in pages):
        raise ValueError("pages and scales are contiguous")
    for name, t, shape in (("block_table", block_table, (batch, block_table.shape[-1])), ("lengths", lengths, (batch,)),
                           ("counts", counts, (batch,))):
        if t is None:
            continue
        if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"{name} is a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    for t in (v, ks, vs, block_table, lengths, counts):
        if t is not None and t.device != k.device:
            raise ValueError(f"pages, block table and lengths are on one device, got {k.device} and {t.device}")


def check_heads(q, k, tables, positions=None) -> None:
    """Shapes of queries and keys (either may be None) and of the rotation's tables."""
    x = k if q is None else q
    if x.dim() != 4 or (q is not None and k is not None and (
            k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3])):
        raise ValueError("queries and keys are [batch, tokens, heads, head_dim] with the same batch, tokens and head_dim")
    cos, sin = tables
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        if (cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape != sin.shape
                or cos.shape[1] * 2 > x.shape[3] or cos.shape[1] < 1):
            raise ValueError("cos and sin are fp32 [positions, rotary_dim / 2] with rotary_dim <= head_dim")
        if positions is not None and (positions.dtype not in (torch.int32, torch.int64) or positions.shape != x.shape[:2]):
            raise ValueError("positions are int32 or int64 [batch, tokens]")
        if positions is None and cos.shape[0] < x.shape[1]:
            raise ValueError(f"tables of {cos.shape[0]} positions are too short for {x.shape[1]} tokens")
    elif positions is not None:
        raise ValueError("positions without cos and sin")


def check_norm_weight(name: str, weight, head_dim: int) -> None:
    if weight is not None and tuple(weight.shape) != (head_dim,):
        raise ValueError(f"{name} has one value per channel of a head, [{head_dim}], got {tuple(weight.shape)}")
