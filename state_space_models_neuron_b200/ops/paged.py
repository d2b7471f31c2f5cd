"""Paged key-value cache: the tensors of one attention layer and what every operation on them checks.

A page holds `page_size` tokens of every key/value head, a head's tokens one behind the other: `k` and `v` are
[pages, kv_heads, page_size, head_dim].  A sequence's token at position p is in slot p % page_size of the page that
`block_table[sequence, p // page_size]` names; sequences share the pool and their pages are in any order.  The head comes before
the token so that the attention kernel reads a head's page as one piece of page_size * head_dim values.

Values are bfloat16, or 8-bit (float8_e4m3fn, int8) with one fp32 scale per token and head in `k_scale` / `v_scale`
[pages, kv_heads, page_size], not negative; a stored value stands for value * scale.
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
    """What holds for every operation on a cache; raises ValueError.  (One expression: a call costs the host as much as its launch.)"""
    k, v, ks, vs = pages
    shape, dtype, dev, i32, f32 = k.shape, k.dtype, k.get_device(), torch.int32, torch.float32
    page = shape[2] if len(shape) == 4 else 0
    if (page >= 16 and not page & (page - 1) and v.shape == shape and v.dtype is dtype and k.is_contiguous() and v.is_contiguous()
            and v.get_device() == dev and block_table.dtype is i32 and block_table.dim() == 2 and block_table.shape[0] == batch
            and block_table.is_contiguous() and block_table.get_device() == dev and lengths.dtype is i32 and lengths.shape == (batch,)
            and lengths.is_contiguous() and lengths.get_device() == dev
            and (counts is None or (counts.dtype is i32 and counts.shape == (batch,) and counts.is_contiguous()
                                    and counts.get_device() == dev))
            and (ks is None and vs is None if dtype not in QUANT_MAX else
                 ks is not None and vs is not None and ks.dtype is f32 and vs.dtype is f32 and ks.shape == shape[:3]
                 and vs.shape == shape[:3] and ks.is_contiguous() and vs.is_contiguous() and ks.get_device() == dev
                 and vs.get_device() == dev)):
        return
    if len(shape) != 4 or v.shape != shape or v.dtype != dtype:
        raise ValueError("k and v pages are [pages, kv_heads, page_size, head_dim] of one shape and type, got "
                         f"{tuple(shape)} {dtype} and {tuple(v.shape)} {v.dtype}")
    if page < 16 or page & (page - 1):
        raise ValueError(f"a page holds a power of two of at least 16 tokens, got {page}")
    if (ks is None) != (vs is None) or (ks is not None) != (dtype in QUANT_MAX):
        raise ValueError("8-bit pages come with scales for keys and values, other pages with none")
    for s in (ks, vs):
        if s is not None and (s.shape != shape[:3] or s.dtype != f32):
            raise ValueError(f"scales are fp32 of shape {tuple(shape[:3])}, got {s.dtype} {tuple(s.shape)}")
    for name, t, wanted in (("block_table", block_table, (batch, block_table.shape[-1])), ("lengths", lengths, (batch,)),
                            ("counts", counts, (batch,))):
        if t is not None and (t.dtype != i32 or tuple(t.shape) != wanted or not t.is_contiguous()):
            raise ValueError(f"{name} is a contiguous int32 tensor of shape {wanted}, got {t.dtype} {tuple(t.shape)}")
    raise ValueError("pages and scales are contiguous and on one device with the block table, lengths and counts")


def check_heads(q, k, cos, sin, positions, from_zero: bool) -> None:
    """Shapes of queries and keys (q may be None) and of the rotation's tables; from_zero: without positions, token l has row l."""
    shape, like = k.shape, k.shape if q is None else q.shape
    if len(shape) != 4 or len(like) != 4 or like[0] != shape[0] or like[1] != shape[1] or like[3] != shape[3]:
        raise ValueError("queries and keys are [batch, tokens, heads, head_dim] with the same batch, tokens and head_dim")
    if shape[2] < 1 or like[2] < 1:
        raise ValueError("queries and keys have at least one head")
    if cos is None and sin is None:
        if positions is not None:
            raise ValueError("positions without cos and sin")
        return
    if cos is None or sin is None:
        raise ValueError("cos and sin come together")
    table = cos.shape
    if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or len(table) != 2 or sin.shape != table
            or not 2 <= table[1] * 2 <= shape[3]):
        raise ValueError("cos and sin are fp32 [positions, rotary_dim / 2] with rotary_dim <= head_dim")
    if positions is not None and (positions.dtype not in (torch.int32, torch.int64) or positions.shape != shape[:2]):
        raise ValueError("positions are int32 or int64 [batch, tokens]")
    if positions is None and from_zero and table[0] < shape[1]:
        raise ValueError(f"tables of {table[0]} positions are too short for {shape[1]} tokens")


def check_norm_weight(name: str, weight, head_dim: int) -> None:
    if weight is not None and weight.shape != (head_dim,):
        raise ValueError(f"{name} has one value per channel of a head, [{head_dim}], got {tuple(weight.shape)}")
