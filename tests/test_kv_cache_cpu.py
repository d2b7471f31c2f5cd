"""Norms of queries and keys with rotation, paged cache and attention of one new token on the CPU: against loops written from the
definitions in 64 bits, gradients against differences, and what the operations refuse."""
import math

import pytest
import torch

from state_space_models_neuron_b200 import ops

EPS = 1e-5


def tables(positions, rotary, theta=10000.0):
    inverse = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inverse
    return angle.cos().float(), angle.sin().float()


def plain_row(x, w, cos, sin):
    """one head's row, channel by channel"""
    x = [float(v) for v in x]
    if w is not None:
        r = 1.0 / math.sqrt(sum(v * v for v in x) / len(x) + EPS)
        x = [v * r * float(g) for v, g in zip(x, w)]
    y = list(x)
    if cos is not None:
        half = len(cos)
        for i in range(half):
            c, s = float(cos[i]), float(sin[i])
            y[i], y[i + half] = x[i] * c - x[i + half] * s, x[i + half] * c + x[i] * s
    return torch.tensor(y, dtype=torch.float64)


@pytest.mark.parametrize("rotary", [0, 4, 8])
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("packed", [True, False])
def test_norm_rotary_is_the_formula(rotary, normed, packed):
    torch.manual_seed(rotary)
    q, k = torch.randn(2, 5, 3, 8, dtype=torch.float64), torch.randn(2, 5, 1, 8, dtype=torch.float64)
    qw, kw = (torch.randn(8, dtype=torch.float64), torch.randn(8, dtype=torch.float64)) if normed else (None, None)
    cos, sin = tables(7, rotary) if rotary else (None, None)
    positions = torch.tensor([[0, 1, 2, 0, 1], [6, 0, 3, 3, 4]], dtype=torch.int32) if packed and rotary else None
    out = ops.qk_norm_rotary(q, k, qw, kw, EPS, cos, sin, positions)
    for x, w, y in zip((q, k), (qw, kw), out):
        for b in range(2):
            for l in range(5):
                p = l if positions is None else int(positions[b, l])
                for h in range(x.shape[2]):
                    ref = plain_row(x[b, l, h], w, *((None, None) if cos is None else (cos[p], sin[p])))
                    torch.testing.assert_close(y[b, l, h], ref, rtol=1e-12, atol=1e-12)


def test_norm_rotary_gradients_are_those_of_differences():
    torch.manual_seed(1)
    args = [torch.randn(1, 3, 2, 8, dtype=torch.float64), torch.randn(1, 3, 1, 8, dtype=torch.float64),
            torch.randn(8, dtype=torch.float64), torch.randn(8, dtype=torch.float64)]
    cos, sin = tables(3, 4)
    args = [a.requires_grad_() for a in args]
    assert torch.autograd.gradcheck(lambda *a: ops.qk_norm_rotary(*a, EPS, cos, sin), args)


def pool(dtype, pages=9, heads=2, page=16, dim=8, fill=None):
    p = ops.kv_pages(pages, heads, page, dim, dtype)
    if fill is not None:
        for t in p:
            if t is not None:
                (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).fill_(fill)
    return p


TABLE = torch.tensor([[3, 7, 0], [8, 1, 2]], dtype=torch.int32)


def at(pages, b, p, which):
    """the value that a cached head row stands for, by the definition of the layout"""
    t, s = (pages.k, pages.k_scale) if which == 0 else (pages.v, pages.v_scale)
    page, slot = int(TABLE[b, p // 16]), p % 16
    x = t[page, :, slot].double()
    return x if s is None else x * s[page, :, slot, None].double()


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("counts", [None, [4, 2]])
def test_write_puts_tokens_where_they_belong(dtype, counts):
    torch.manual_seed(2)
    k, v, q = torch.randn(2, 5, 2, 8), torch.randn(2, 5, 2, 8), torch.randn(2, 5, 4, 8)
    kw, qw = torch.rand(8) + 0.5, torch.rand(8) + 0.5
    cos, sin = tables(48, 4)
    pages = pool(dtype)
    before = [None if t is None else t.clone() for t in pages]
    lengths = torch.tensor([18, 3], dtype=torch.int32)                 # the second sequence: 5 given tokens begin at -2
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    out = ops.kv_cache_write(k, v, pages, TABLE, lengths, counts=c, q=q, q_weight=qw, k_weight=kw, eps=EPS, cos=cos, sin=sin)
    written = set()
    # half a step of the type: bf16 2^-8, e4m3 2^-4 of the value and half of its smallest step 2^-9 of the scale (row maximum / 448);
    # int8 half a step, which is the row maximum / 127; each with the fp32 steps in front
    step = {torch.float64: 0, torch.bfloat16: 2 ** -8, torch.float8_e4m3fn: 2 ** -4, torch.int8: 0}[dtype] + 2 ** -20
    floor = {torch.float64: 0, torch.bfloat16: 0, torch.float8_e4m3fn: 2 ** -10 / 448, torch.int8: 0.5 / 127}[dtype]
    for b in range(2):
        n = 5 if counts is None else counts[b]
        for l in range(5):
            p = int(lengths[b]) - n + l
            if l >= n or p < 0:
                assert not out[b, l].any()
                continue
            written.add((int(TABLE[b, p // 16]), p % 16))
            for h in range(4):
                torch.testing.assert_close(out[b, l, h].double(), plain_row(q[b, l, h], qw, cos[p], sin[p]), rtol=1e-5, atol=1e-5)
            for which, ref in ((0, torch.stack([plain_row(k[b, l, h], kw, cos[p], sin[p]) for h in range(2)])), (1, v[b, l].double())):
                far = (at(pages, b, p, which) - ref).abs()
                assert (far <= step * ref.abs() + (floor * (1 + 2 ** -18) + 2 ** -20) * ref.abs().amax(-1, keepdim=True)).all()
    # everything else is as it was
    for t, old in zip(pages, before):
        if t is not None:
            for page in range(9):
                for slot in range(16):
                    if (page, slot) not in written:
                        assert torch.equal(t[page, :, slot].float(), old[page, :, slot].float())


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_rows_of_zeros_of_tiny_and_of_non_finite_values(dtype):
    x = torch.zeros(1, 4, 1, 8)
    x[0, 1] = 1e-38
    x[0, 2, 0, 3] = math.inf
    x[0, 3, 0, 0] = math.nan
    pages = pool(dtype, heads=1)
    ops.kv_cache_write(x, x, pages, TABLE[:1], torch.tensor([4], dtype=torch.int32))
    k, v = ops.kv_cache_read(pages, TABLE[:1], torch.tensor([4], dtype=torch.int32), 6, torch.float32)
    for t in (k, v):
        assert not t[0, :2].any() and t[0, 2:4].isnan().all() and not t[0, 4:].any()


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16, torch.float8_e4m3fn, torch.int8])
def test_attention_is_the_formula(dtype):
    torch.manual_seed(3)
    pages = pool(dtype)
    lengths = torch.tensor([37, 0], dtype=torch.int32)
    if dtype not in (torch.float64,):
        # what lies behind the lengths is never used
        for t in pages:
            if t is not None and t.dtype != torch.int8:
                (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).fill_(0x7f if t.dtype == torch.float8_e4m3fn else math.nan)
    k, v = torch.randn(2, 37, 2, 8), torch.randn(2, 37, 2, 8)
    ops.kv_cache_write(k[:1], v[:1], pages, TABLE[:1], lengths[:1])
    q = torch.randn(2, 1, 6, 8, dtype=torch.float64)
    out = ops.paged_attention(q, pages, TABLE, lengths)
    assert not out[1].any()
    for h in range(6):
        s = [float((q[0, 0, h] * at(pages, 0, p, 0)[h // 3]).sum()) / math.sqrt(8) for p in range(37)]
        e = [math.exp(x - max(s)) for x in s]
        ref = sum(x * at(pages, 0, p, 1)[h // 3] for p, x in enumerate(e)) / sum(e)
        torch.testing.assert_close(out[0, 0, h], ref, rtol=1e-5, atol=1e-5)
    rk, rv = ops.kv_cache_read(pages, TABLE, lengths, 40, torch.float32)
    for p in range(37):
        torch.testing.assert_close(rk[0, p].double(), at(pages, 0, p, 0), rtol=1e-6, atol=0)
        torch.testing.assert_close(rv[0, p].double(), at(pages, 0, p, 1), rtol=1e-6, atol=0)
    assert not rk[0, 37:].any() and not rk[1].any() and not rv[1].any()


def refusals(device, q, k, pages, table, lengths, cos, sin, w):
    """(error, call) of what every device refuses"""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    B, L, H, D = q.shape
    one = q[:, :1]
    write = lambda **kw: ops.kv_cache_write(**{**dict(k=k, v=k, pages=pages, block_table=table, lengths=lengths), **kw})  # noqa: E731
    return [
        (ValueError, lambda: ops.qk_norm_rotary(q[0], k, w, w, EPS)),
        (ValueError, lambda: ops.qk_norm_rotary(q, k[:, 1:], w, w, EPS)),
        (ValueError, lambda: ops.qk_norm_rotary(q, k[..., :-16], w, w, EPS)),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w[:-1], w, EPS)),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w[:1], EPS)),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w, EPS, cos, None)),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w, EPS, cos.double(), sin.double())),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w, EPS, cos[:L - 1], sin[:L - 1])),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w, EPS, torch.cat([cos] * 9, 1), torch.cat([sin] * 9, 1))),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w, EPS, positions=torch.zeros(B, L, dtype=torch.int32, device=device))),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w, EPS, cos, sin, torch.zeros(B, L, device=device))),
        (ValueError, lambda: ops.qk_norm_rotary(q, k, w, w, EPS, cos, sin, torch.zeros(B, L + 1, dtype=torch.int64, device=device))),
        (ValueError, lambda: write(v=k[:, :, :1])),
        (ValueError, lambda: write(v=k.double())),
        (ValueError, lambda: write(q=q[:, 1:])),
        (ValueError, lambda: write(lengths=lengths.long())),
        (ValueError, lambda: write(lengths=lengths[:1])),
        (ValueError, lambda: write(block_table=table.long())),
        (ValueError, lambda: write(block_table=table[:1])),
        (ValueError, lambda: write(block_table=table.t().contiguous().t())),
        (ValueError, lambda: write(counts=i32(1, 1, 1))),
        (ValueError, lambda: write(k_weight=w[:-1])),
        (ValueError, lambda: write(cos=cos)),
        (ValueError, lambda: write(pages=ops.KVPages(pages.k, pages.v[1:]))),
        (ValueError, lambda: write(pages=ops.KVPages(pages.k[:, :1], pages.v[:, :1]))),
        (ValueError, lambda: write(pages=ops.KVPages(pages.k, pages.v, *(torch.zeros(pages.k.shape[:3], device=device),) * 2))),
        (ValueError, lambda: write(pages=ops.kv_pages(4, k.shape[2], 8, D, torch.bfloat16, device))),
        (ValueError, lambda: write(pages=ops.kv_pages(4, k.shape[2], 48, D, torch.bfloat16, device))),
        (ValueError, lambda: write(pages=ops.kv_pages(4, k.shape[2], 16, D // 2, torch.bfloat16, device))),
        (ValueError, lambda: ops.kv_cache_write(k, k, ops.KVPages(pages.k.to(torch.int8), pages.v.to(torch.int8)), table, lengths)),
        (ValueError, lambda: ops.kv_cache_read(pages, table, lengths, -1)),
        (ValueError, lambda: ops.kv_cache_read(pages, table, lengths[:1], 4)),
        (ValueError, lambda: ops.paged_attention(q, pages, table, lengths)),
        (ValueError, lambda: ops.paged_attention(one[:, :, :H - 1], pages, table, lengths)),
        (ValueError, lambda: ops.paged_attention(one[..., :-16], pages, table, lengths)),
        (ValueError, lambda: ops.paged_attention(one, pages, table, lengths.float())),
        (ValueError, lambda: ops.paged_attention(one[:1], pages, table, lengths)),
    ]


def test_refusals():
    q, k, w = torch.randn(2, 5, 4, 32), torch.randn(2, 5, 2, 32), torch.ones(32)
    pages = ops.kv_pages(9, 2, 16, 32, torch.float32)
    lengths = torch.tensor([18, 20], dtype=torch.int32)
    cos, sin = tables(48, 8)
    for n, (error, call) in enumerate(refusals("cpu", q, k, pages, TABLE, lengths, cos, sin, w)):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {n} was not refused")


def test_values_that_only_the_data_shows_are_refused():
    q, k = torch.randn(2, 5, 4, 32), torch.randn(2, 5, 2, 32)
    pages = ops.kv_pages(9, 2, 16, 32, torch.float32)
    cos, sin = tables(48, 8)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    fine = dict(k=k, v=k, pages=pages, block_table=TABLE, lengths=i32(18, 20))
    for change in (dict(lengths=i32(18, 49)), dict(block_table=TABLE + 1), dict(block_table=TABLE - 9), dict(counts=i32(1, 6)),
                   dict(counts=i32(-1, 3)), dict(cos=cos[:19], sin=sin[:19])):
        with pytest.raises(ValueError):
            ops.kv_cache_write(**{**fine, **change})
            pytest.fail(f"{change} was not refused")
    assert not pages.k.any() and not pages.v.any()
    for table, lengths in ((TABLE, i32(18, 49)), (TABLE + 1, i32(18, 20)), (TABLE - 9, i32(18, 20))):
        with pytest.raises(ValueError):
            ops.kv_cache_read(pages, table, lengths, 60)
        with pytest.raises(ValueError):
            ops.paged_attention(q[:, :1], pages, table, lengths)
    for bad in (48, -1):
        with pytest.raises(ValueError):
            ops.qk_norm_rotary(q, k, None, None, EPS, cos, sin, torch.full((2, 5), bad))


def test_empty_batches_and_prompts():
    pages = ops.kv_pages(9, 2, 16, 32, torch.float32)
    none = torch.zeros(0, dtype=torch.int32)
    assert ops.kv_cache_write(torch.zeros(0, 3, 2, 32), torch.zeros(0, 3, 2, 32), pages, TABLE[:0], none) is None
    assert ops.kv_cache_write(torch.zeros(2, 0, 2, 32), torch.zeros(2, 0, 2, 32), pages, TABLE, none.new_zeros(2),
                              q=torch.zeros(2, 0, 4, 32)).shape == (2, 0, 4, 32)
    assert ops.paged_attention(torch.zeros(0, 1, 4, 32), pages, TABLE[:0], none).shape == (0, 1, 4, 32)
    assert ops.kv_cache_read(pages, TABLE, none.new_zeros(2), 0)[0].shape == (2, 0, 2, 32)
    assert ops.qk_norm_rotary(torch.zeros(2, 0, 4, 32), torch.zeros(2, 0, 2, 32), None, None, EPS)[0].shape == (2, 0, 4, 32)
