"""Paged key-value cache and attention of one new token on the GPU, against the definitions in 64 bits."""
import math

import pytest
import torch

from state_space_models_neuron_b200 import ops
from tests.test_gpu_qk_norm import tables, turned
from tests.test_kv_cache_cpu import refusals

pytestmark = pytest.mark.gpu
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
U16 = 2.0 ** -8


@pytest.fixture(autouse=True)
def _status():
    yield
    from state_space_models_neuron_b200.ops import cuda_ops
    torch.cuda.synchronize()
    cuda_ops.check_status()


def make_pool(B, width, heads, page, dim, dtype, seed=0, spare=3):
    """zeroed pages and a table of pages in random order"""
    g = torch.Generator().manual_seed(seed)
    n = B * width + spare
    table = torch.randperm(n, generator=g)[:B * width].view(B, width).to(torch.int32).cuda()
    return ops.kv_pages(n, heads, page, dim, dtype, "cuda"), table


def poison(pages):
    """stale contents that no result may depend on: NaN where the type has it, the largest value elsewhere"""
    for t in pages:
        if t is None:
            continue
        if t.dtype == torch.int8:
            t.fill_(127)
        elif t.dtype == torch.float8_e4m3fn:
            t.view(torch.uint8).fill_(0x7f)
        else:
            t.fill_(math.nan)


def stands_for(pages, table, b, n):
    """keys and values of the first n tokens of sequence b in 64 bits, [n, heads, dim]"""
    page = pages.k.shape[2]
    at = torch.arange(n, device="cuda")
    ids, slot = table[b].long()[at // page], at % page
    out = []
    for t, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        raw = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        x = raw[ids, :, slot]
        x = (x.view(t.dtype) if t.dtype == torch.float8_e4m3fn else x).double()
        out.append(x if s is None else x * s[ids, :, slot][..., None].double())
    return out


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def draw(shape, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g) * torch.empty(shape[-1], device="cuda").log_normal_(0, 0.5, generator=g)
    return (x * size).bfloat16()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,Hq,Hk,D,rotary,page,lengths,counts", [
    (1, 32, 8, 128, 128, 16, (1, 16, 17, 200), None),              # one token: first, last and first slot of a page
    (1, 5, 1, 64, 32, 64, (0, 1, 64, 65), None),                   # an idle sequence
    (37, 9, 3, 128, 0, 16, (37, 100, 20, 5), None),                # the last two padded on the left
    (50, 4, 2, 256, 256, 32, (50, 70, 9, 0), (50, 13, 9, 0)),      # padded on the right
    (130, 2, 2, 64, 16, 256, (130, 131, 386, 1), (130, 1, 129, 1)),
])
@pytest.mark.parametrize("normed", [True, False])
def test_write_and_read(dtype, L, Hq, Hk, D, rotary, page, lengths, counts, normed):
    dtype, B = TYPES[dtype], len(lengths)
    width = -(-max(lengths) // page) + 1
    pages, table = make_pool(B, width, Hk, page, D, dtype, seed=L)
    poison(pages)
    before = [None if t is None else t.clone() for t in pages]
    qkv = draw((B, L, Hq + 2 * Hk, D), L + D)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    qw, kw = ((1 + 0.2 * draw((D,), 3)).bfloat16(), (1 + 0.2 * draw((D,), 4)).float()) if normed else (None, None)
    cos, sin = tables(max(lengths) + 2, rotary) if rotary else (None, None)
    n, c = ints(*lengths), None if counts is None else ints(*counts)
    out = ops.kv_cache_write(k, v, pages, table, n, counts=c, q=q, q_weight=qw, k_weight=kw, eps=EPS, cos=cos, sin=sin)
    got = ops.kv_cache_read(pages, table, n, width * page, torch.float32)
    half = ops.kv_cache_read(pages, table, n, max(lengths), torch.bfloat16)
    touched = torch.zeros(pages.k.shape[0], page, dtype=torch.bool, device="cuda")
    for b in range(B):
        count = L if counts is None else counts[b]
        first = max(0, count - lengths[b])                          # tokens in front of position 0
        new = slice(first, count)
        at = torch.arange(lengths[b] - count + first, lengths[b], device="cuda")[None]
        touched[table[b].long()[at[0] // page], at[0] % page] = True
        assert not out[b, :first].any() and not out[b, count:].any()
        if count == first:
            continue
        for x, w, y, rotates in ((q, qw, out[b, new], True), (k, kw, got[0][b, at[0]], True), (v, None, got[1][b, at[0]], False)):
            x = x[b:b + 1, new].double()
            if w is not None:
                x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
            ref = (turned(x, cos, sin, at) if rotates else x)[0]
            size = x[0].abs().amax(-1, keepdim=True)
            # steps in front as in the norm's own test, 2^-18; then half a step of what holds it: bf16 2^-8; e4m3 2^-4 and half its
            # smallest step, 2^-10 of the scale; int8 half the scale (row maximum / 448, / 127)
            if y.dtype == torch.bfloat16 or dtype == torch.bfloat16:
                bound = 2 ** -8 * ref.abs()
            elif dtype == torch.float8_e4m3fn:
                bound = 2 ** -4 * ref.abs() + 2 ** -10 / 448 * ref.abs().amax(-1, keepdim=True)
            else:
                bound = 0.5 / 127 * ref.abs().amax(-1, keepdim=True)
            assert ((y.double() - ref).abs() <= bound * (1 + 2 ** -17) + 2 ** -17 * size).all()
    # every row that was read, against what the pages hold: one fp32 product, one rounding
    for b in range(B):
        held = stands_for(pages, table, b, max(0, lengths[b]))
        for x, wide, narrow in zip(held, (got[0][b], got[1][b]), (half[0][b], half[1][b])):
            m = x.shape[0]
            real = ~x.isnan().any(-1, keepdim=True).expand_as(x)   # tokens that were there before are poison
            assert ((wide[:m].double() - x).abs() <= 2 ** -24 * x.abs())[real].all()
            assert ((narrow[:m].double() - x).abs() <= (2 ** -8 + 2 ** -23) * x.abs())[real].all()
            assert not wide[m:].any() and not narrow[m:].any()
    # and nothing else was written
    for t, old in zip(pages, before):
        if t is not None:
            same = (t.view(torch.uint8) == old.view(torch.uint8)).view(*t.shape[:3], -1).all(-1)
            assert same.transpose(1, 2)[~touched].all()


def attention_bound(q, k, v, scale, lost=2 ** -24):
    """(result, bound) for one sequence in 64 bits: q [Hq, D], k / v [n, Hk, D].
    bound: an fp32 score is a sum of D products (at most D + 8 roundings), its exponential takes 2^-22 of the exponent more; the
    probabilities may be rounded to bf16 before they meet the values (2^-8 each); the result is rounded to bf16.
    Beside 8-bit values a probability may be held in fp16, with its value's scale, as a share of a number that is at most twice the
    largest such product (a power of two): fp16 steps by 2^-24 below 2^-14, so a share is off by at most half of that, 2^-25 (one below it may
    vanish), and n of them by n 2^-24 max_t(p_t max_c |v_tc|).  That can be all of a channel in which the one token with a large share holds a zero.  bf16 and
    fp32 go down to 2^-126 (lost).  An fp32 product of probability and scale below 2^-126 is flushed to zero; a stored value is at
    most 448, so each token that does not hold zeros alone is off by at most 448 * 2^-126 (1e-35) by that."""
    n, Hk, D = k.shape
    qg = q.view(Hk, -1, D)
    s = torch.einsum("kgd,tkd->kgt", qg, k) * scale
    size = torch.einsum("kgd,tkd->kgt", qg.abs(), k.abs()).amax(-1, keepdim=True) * scale
    off = (D + 8) * 2 ** -24 * size + 2 ** -21 * s.abs().amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    ref = torch.einsum("kgt,tkd->kgd", p, v)
    mass = torch.einsum("kgt,tkd->kgd", p, v.abs())
    # the values' sum over n tokens in fp32, with 2^-17 for its roundings
    largest = (p * v.abs().amax(-1).t()[:, None]).amax(-1, keepdim=True)
    bound = U16 * ref.abs() + mass * (U16 + 2 * off + 2 ** -17) + n * lost * largest + 448 * 2 ** -126 * v.any(-1).sum(0).view(Hk, 1, 1)
    return ref.reshape(-1, D), bound.reshape(-1, D)


def check_attention(q, pages, table, lengths, out, scale=None):
    D = q.shape[-1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    for b, n in enumerate(lengths):
        if n <= 0:
            assert not out[b].any()
            continue
        k, v = stands_for(pages, table, b, n)
        ref, bound = attention_bound(q[b, 0].double(), k, v, scale, 2 ** -126 if pages.k_scale is None else 2 ** -24)
        far = (out[b, 0].double() - ref).abs()
        assert (far <= bound).all(), (b, n, (far - bound).max().item(), (far / bound).max().item())


def filled(B, lengths, Hk, D, page, dtype, seed, size=1.0):
    width = max(1, -(-max(lengths) // page))
    pages, table = make_pool(B, width, Hk, page, D, dtype, seed)
    poison(pages)
    L = max(1, max(lengths))
    ops.kv_cache_write(draw((B, L, Hk, D), seed + 1, size), draw((B, L, Hk, D), seed + 2), pages, table, ints(*lengths),
                       counts=ints(*[max(0, n) for n in lengths]))
    return pages, table


RAGGED = (1, 15, 0, 16, 17, 31, 33, 64, 127, 128, 500, -1, 1025)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (4, 1), (8, 1), (9, 3), (16, 1), (32, 8), (20, 2), (40, 2), (7, 7)])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 128), (256, 32)])
def test_attention(dtype, Hq, Hk, D, page):
    pages, table = filled(len(RAGGED), RAGGED, Hk, D, page, TYPES[dtype], Hq + D)
    q = draw((len(RAGGED), 1, Hq, D), 5, 2.0)
    check_attention(q, pages, table, RAGGED, ops.paged_attention(q, pages, table, ints(*RAGGED)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [(1,), (20000,), (3, 12345), (4096, 4095, 4097), (777,) * 70, (1,) * 300, (3000, 100) * 30, (9000,) + (1,) * 40])
def test_attention_over_lengths_and_batches(dtype, lengths):
    pages, table = filled(len(lengths), lengths, 2, 128, 64, TYPES[dtype], 11)
    q = draw((len(lengths), 1, 8, 128), 6, 1.5)
    check_attention(q, pages, table, lengths, ops.paged_attention(q, pages, table, ints(*lengths)))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_to_sharp_and_to_far_tokens(dtype):
    """large scores of both signs: one token takes nearly all, first, last or in the middle; queries that are zero or tiny; a scale"""
    lengths = (700, 700, 700, 700, 700, 700)
    pages, table = filled(6, lengths, 2, 128, 32, TYPES[dtype], 13, size=4.0)
    k, _ = ops.kv_cache_read(pages, table, ints(*lengths), 700)
    q = torch.stack([k[0, 0], k[1, 699], k[2, 350], -k[3, 10], torch.zeros_like(k[4, 0]), k[5, 5] * 2 ** -40])
    q = q[:, None].repeat_interleave(3, 2).contiguous()
    check_attention(q, pages, table, lengths, ops.paged_attention(q, pages, table, ints(*lengths)))
    check_attention(q, pages, table, lengths, ops.paged_attention(q, pages, table, ints(*lengths), scale=0.7), 0.7)
    check_attention(q, pages, table, lengths, ops.paged_attention(q, pages, table, ints(*lengths), scale=0.0), 0.0)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_attention_with_scales_far_apart(dtype):
    """values of tokens that differ by 2^60: what a probability loses against the largest must not be lost to the sum"""
    pages, table = filled(2, (300, 90), 2, 128, 16, TYPES[dtype], 17)
    g = torch.Generator(device="cuda").manual_seed(3)
    power = torch.randint(-60, 1, pages.v_scale.shape, device="cuda", generator=g).float()
    pages.v_scale.copy_(torch.where(pages.v_scale.isnan(), pages.v_scale, pages.v_scale * torch.exp2(power)))
    q = draw((2, 1, 8, 128), 7, 3.0)
    check_attention(q, pages, table, (300, 90), ops.paged_attention(q, pages, table, ints(300, 90)))
    # one token holds all: the others' values are zero
    pages.v_scale.fill_(0.0)
    pages.v_scale[table[0, 3].item(), :, 5] = 1e-30
    check_attention(q, pages, table, (300, 90), ops.paged_attention(q, pages, table, ints(300, 90)))


def test_attention_with_values_that_are_not_finite():
    """NaN and infinity inside a sequence reach its heads and no others"""
    pages, table = filled(3, (40, 50, 60), 2, 64, 16, torch.bfloat16, 19)
    q = draw((3, 1, 4, 64), 8)
    good = ops.paged_attention(q, pages, table, ints(40, 50, 60))
    pages.k[table[1, 1].item(), 0, 2, 5] = math.nan
    pages.v[table[2, 2].item(), 1, 1, 7] = math.inf
    out = ops.paged_attention(q, pages, table, ints(40, 50, 60))
    assert out[1, 0, :2].isnan().all() and torch.equal(out[1, 0, 2:], good[1, 0, 2:]) and torch.equal(out[0], good[0])
    assert torch.equal(out[2, 0, :2], good[2, 0, :2])
    assert (out[2, 0, 2:, 7] == math.inf).all()
    rest = torch.arange(64, device="cuda") != 7
    assert torch.equal(out[2, 0, 2:][:, rest], good[2, 0, 2:][:, rest])


def test_query_layouts():
    pages, table = filled(3, (40, 50, 60), 2, 128, 16, torch.bfloat16, 23)
    n = ints(40, 50, 60)
    q = draw((3, 1, 8, 128), 9)
    good = ops.paged_attention(q, pages, table, n)
    big = draw((3, 1, 12, 128), 10)
    big[:, :, 2:10] = q
    odd = torch.zeros(3, 1, 8, 129, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = q
    for same in (big[:, :, 2:10], odd[..., 1:], q.transpose(0, 2).contiguous().transpose(0, 2)):
        assert torch.equal(ops.paged_attention(same, pages, table, n), good)
    # a pool of several layers: its pages are views
    both = [torch.stack([torch.zeros_like(t), t]) for t in (pages.k, pages.v)]
    assert torch.equal(ops.paged_attention(q, ops.KVPages(both[0][1], both[1][1]), table, n), good)
    # shared pages: two sequences with the same prompt
    shared = ops.paged_attention(q[:1].expand(2, -1, -1, -1), pages, table[:1].expand(2, -1).contiguous(), ints(40, 40))
    assert torch.equal(shared[0], good[0]) and torch.equal(shared[1], good[0])


@pytest.mark.parametrize("lengths", [(5000, 1, 777, 20000), (200, 37) * 60, (2000, 2500) * 20])
def test_runs_give_the_same_bits(lengths):
    pages, table = filled(len(lengths), lengths, 2, 128, 64, torch.bfloat16, 29)
    q = draw((len(lengths), 1, 8, 128), 12)
    first = ops.paged_attention(q, pages, table, ints(*lengths))
    for _ in range(20):
        assert torch.equal(ops.paged_attention(q, pages, table, ints(*lengths)), first)


def test_pages_beyond_two_to_the_31_values():
    page, D = 256, 128
    n = 2 ** 31 // (page * D) + 20
    k = torch.zeros(n, 1, page, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    pages, table = ops.KVPages(k, v), ints(n - 2, n - 1)[None].contiguous()
    lengths = (400,)
    x, y = draw((1, 400, 1, D), 14), draw((1, 400, 1, D), 15)
    ops.kv_cache_write(x, y, pages, table, ints(*lengths))
    got = ops.kv_cache_read(pages, table, ints(*lengths), 400)
    assert torch.equal(got[0], x) and torch.equal(got[1], y)
    q = draw((1, 1, 4, D), 16)
    check_attention(q, pages, table, lengths, ops.paged_attention(q, pages, table, ints(*lengths)))


@pytest.mark.parametrize("dtype", TYPES)
def test_bad_pages_are_skipped_and_reported(dtype):
    from state_space_models_neuron_b200.ops import cuda_ops

    def reported():
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="status 3"):
            cuda_ops.check_status()

    lengths = (60, 60)
    pages, table = filled(2, lengths, 2, 64, 16, TYPES[dtype], 31)
    q, n = draw((2, 1, 4, 64), 17), ints(*lengths)
    good = ops.paged_attention(q, pages, table, n)
    held = [t.clone() for t in pages if t is not None]
    x = draw((2, 3, 2, 64), 18)
    for value in (-1, pages.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        bad = table.clone()
        bad[1, 3] = value                                              # the last page of the second sequence
        out = ops.paged_attention(q, pages, bad, n)
        reported()
        assert torch.equal(out[0], good[0])
        k, v = (t[:48] for t in stands_for(pages, table, 1, 60))
        ref, bound = attention_bound(q[1, 0].double(), k, v, 0.125)
        assert ((out[1, 0].double() - ref).abs() <= bound).all()
        read = ops.kv_cache_read(pages, bad, n, 60)
        reported()
        assert not read[0][1, 48:].any() and not read[1][1, 48:].any() and read[0][1, :48].any()
        assert ops.kv_cache_write(x[1:], x[1:], pages, bad[1:], n[1:], q=x[1:])[0].any().item() is False
        reported()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held, [t for t in pages if t is not None]))
    # lengths behind the table, counts outside, tables too short
    out = ops.paged_attention(q, pages, table, ints(60, 10 ** 9))
    reported()
    assert torch.equal(out[0], good[0])
    ops.kv_cache_read(pages, table, ints(60, 2 ** 31 - 1), 70)
    reported()
    for change in (dict(lengths=ints(60, 10 ** 9)), dict(counts=ints(3, 4), lengths=ints(60, 2)), dict(counts=ints(3, -1))):
        ops.kv_cache_write(**{**dict(k=x, v=x, pages=pages, block_table=table, lengths=n), **change})
        reported()
    cos, sin = tables(59, 64)
    ops.kv_cache_write(x, x, pages, table, n, cos=cos, sin=sin)
    reported()


def test_refusals():
    q, k, w = draw((2, 5, 4, 128), 1), draw((2, 5, 2, 128), 2), torch.ones(128, device="cuda")
    pages, table = make_pool(2, 3, 2, 16, 128, torch.bfloat16)
    n = ints(18, 20)
    cos, sin = tables(48, 32)
    one = q[:, :1]
    more = [
        (TypeError, lambda: ops.kv_cache_write(k.float(), k.float(), pages, table, n)),
        (TypeError, lambda: ops.kv_cache_write(k, k, pages, table, n, q=q.half())),
        (TypeError, lambda: ops.kv_cache_write(k, k, pages, table, n, k_weight=w.half())),
        (TypeError, lambda: ops.kv_cache_write(k, k, ops.KVPages(pages.k.half(), pages.v.half()), table, n)),
        (TypeError, lambda: ops.kv_cache_read(pages, table, n, 4, torch.float16)),
        (TypeError, lambda: ops.paged_attention(one.float(), pages, table, n)),
        (TypeError, lambda: ops.paged_attention(one, ops.KVPages(pages.k.float(), pages.v.float()), table, n)),
        (ValueError, lambda: ops.kv_cache_write(k, k, pages, table, n.cpu())),
        (ValueError, lambda: ops.kv_cache_write(k, k, pages, table, n, cos=tables(48, 24)[0], sin=tables(48, 24)[1])),
        (ValueError, lambda: ops.kv_cache_write(k, k, pages, table, n, cos=cos.cpu(), sin=sin.cpu())),
        (ValueError, lambda: ops.kv_cache_write(k, k, ops.KVPages(pages.k.cpu(), pages.v.cpu()), table, n)),
        (ValueError, lambda: ops.paged_attention(one, pages, table.cpu(), n)),
        (ValueError, lambda: ops.paged_attention(one[..., :32], ops.kv_pages(9, 2, 16, 32, torch.bfloat16, "cuda"), table, n)),
    ]
    for i, (error, call) in enumerate(refusals("cuda", q, k, pages, table, n, cos, sin, w) + more):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was not refused")
    ops.kv_cache_write(k, k, pages, table, n)                          # and the plain call is none of them


def test_empty_batches_and_prompts():
    pages, table = make_pool(2, 3, 2, 16, 128, torch.bfloat16)
    none = ints(0, 0)
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    assert ops.kv_cache_write(z(0, 3, 2, 128), z(0, 3, 2, 128), pages, table[:0], none[:0]) is None
    assert ops.kv_cache_write(z(2, 0, 2, 128), z(2, 0, 2, 128), pages, table, none, q=z(2, 0, 4, 128)).shape == (2, 0, 4, 128)
    assert ops.paged_attention(z(0, 1, 4, 128), pages, table[:0], none[:0]).shape == (0, 1, 4, 128)
    assert not ops.paged_attention(z(2, 1, 4, 128) + 1, pages, table[:, :0].contiguous(), none).any()
    assert ops.kv_cache_read(pages, table, none, 0)[0].shape == (2, 0, 2, 128)
    assert ops.qk_norm_rotary(z(2, 0, 4, 128), z(2, 0, 2, 128), None, None, EPS)[0].shape == (2, 0, 4, 128)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_one_by_one_captured_and_on_two_streams(dtype):
    """write and attend as a decoding layer does: eagerly, from a replayed graph, and by two graphs at once on two streams"""
    B, Hq, Hk, D, page, start, steps = 3, 8, 2, 128, 16, 30, 5
    dtype = TYPES[dtype]
    cos, sin = tables(64, 128)
    w = torch.ones(D, device="cuda")
    tokens = [draw((B, 1, Hq + 2 * Hk, D), 100 + i) for i in range(steps)]

    def fresh():
        pages, table = filled(B, (start,) * B, Hk, D, page, dtype, 41)
        wide = torch.cat([table, torch.zeros(B, 1, dtype=torch.int32, device="cuda")], 1)
        more = ops.KVPages(*[None if t is None else torch.cat([t, torch.zeros_like(t[:B])]) for t in pages])
        wide[:, -1] = torch.arange(B, device="cuda") + pages.k.shape[0]
        return more, wide, torch.full((B,), start, dtype=torch.int32, device="cuda")

    def token(x, pages, table, n):
        n += 1
        q = ops.kv_cache_write(x[:, :, Hq:Hq + Hk], x[:, :, Hq + Hk:], pages, table, n, q=x[:, :, :Hq], q_weight=w, k_weight=w, eps=EPS,
                               cos=cos, sin=sin)
        return ops.paged_attention(q, pages, table, n)

    state = fresh()
    eager = []
    for x in tokens:
        eager.append(token(x, *state))
    check_attention(ops.qk_norm_rotary(tokens[-1][:, :, :Hq], tokens[-1][:, :, Hq:Hq + Hk], w, w, EPS, cos, sin,
                                       torch.full((B, 1), start + steps - 1, device="cuda"))[0],
                    state[0], state[1], [start + steps] * B, eager[-1])
    graphs = []
    for _ in range(2):
        state = fresh()
        static = tokens[0].clone()
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            token(static, *fresh())
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            out = token(static, *state)
        graphs.append((graph, static, out, side, state))
    torch.cuda.synchronize()
    for i, x in enumerate(tokens):
        for graph, static, out, side, _ in graphs:
            with torch.cuda.stream(side):
                static.copy_(x)
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, _, _ in graphs:
            assert torch.equal(out, eager[i])


def test_writing_tells_autograd():
    pages, table = make_pool(1, 2, 1, 16, 64, torch.bfloat16)
    x = draw((1, 3, 1, 64), 1)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    kept = (pages.k[0, 0] * w).sum()
    ops.kv_cache_write(x, x, pages, table, ints(3))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
