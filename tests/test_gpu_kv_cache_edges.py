"""Paged key-value cache on the GPU where rounding, schedules and failures meet their edges."""
import pytest
import torch

from state_space_models_neuron_b200 import ops
from tests.test_gpu_kv_cache import TYPES, check_attention, draw, filled, ints, make_pool, stands_for

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    from state_space_models_neuron_b200.ops import cuda_ops
    torch.cuda.synchronize()
    cuda_ops.check_status()


def same_bits(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_stored_bytes_are_those_of_the_definition(dtype, D):
    """scale = max |x| / Qmax and x / scale rounded to nearest even, each as fp32 division and rounding give it on the CPU: rows of
    every mantissa and of large and small exponents, with values half of the maximum and other ties"""
    g = torch.Generator().manual_seed(D)
    n = 4096
    top = (1 + torch.arange(n) % 128 / 128) * torch.exp2(torch.randint(-99, 127, (n,), generator=g).float())
    part = torch.rand(n, D, generator=g) * torch.exp2(-torch.randint(0, 14, (n, D), generator=g).float())
    part[:, 0] = 1
    part[:, 1:D // 4] = 0.5                                           # 63.5 of 127: between two integers
    part[:, D // 4:D // 2] = (torch.randint(0, 448, (n, D // 4), generator=g) + 0.5) / 448
    x = (top[:, None] * part * (1 - 2 * torch.randint(0, 2, (n, D), generator=g))).bfloat16().view(4, n // 8, 2, D)
    made = {}
    for device in ("cpu", "cuda"):
        pages, table = make_pool(4, n // 8 // 64, 2, 64, D, TYPES[dtype], seed=1)
        pages, table = ops.KVPages(*(t.to(device) for t in pages)), table.to(device)
        ops.kv_cache_write(x.to(device), (-x).to(device), pages, table, ints(*[n // 8] * 4).to(device))
        made[device] = pages
    for a, b in zip(made["cuda"], made["cpu"]):
        assert same_bits(a, b)


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("Hq", [8, 32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("far", [10, 20, 28])
def test_queries_beside_much_larger_ones(dtype, Hq, D, far):
    """one channel of a query is 2^far larger than the others, and its keys are zero: the others decide alone"""
    lengths = (100, 333)
    pages, table = filled(2, lengths, 2, D, 16, TYPES[dtype], far)
    pages.k.view(torch.uint8)[..., D // 3] = 0
    q = draw((2, 1, Hq, D), D, 1.5)
    q[..., D // 3] = 1.25 * 2 ** far
    check_attention(q, pages, table, lengths, ops.paged_attention(q, pages, table, ints(*lengths)))


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("power", [-126, -100, 100, 110])
def test_queries_of_every_size(dtype, power):
    """queries of 2^power beside keys of about 2^-power, bf16's smallest numbers (2^-126 and below it) included"""
    lengths = (100, 333)
    pages, table = filled(2, lengths, 2, 128, 16, TYPES[dtype], 3)
    pages.k_scale.copy_((pages.k_scale.double() * 2.0 ** -power).float())
    q = (draw((2, 1, 16, 128), 4).double() * 2.0 ** power).bfloat16()
    check_attention(q, pages, table, lengths, ops.paged_attention(q, pages, table, ints(*lengths)))


def tight_bound(q, k, v, scale, v_scale=None):
    """(result, bound) of one sequence in 64 bits, with what the kernel claims (v_scale [n, Hk]: of 8-bit values).

    Scores are fp32 sums of D products (D + 8 roundings), exponentials are good to 2^-22 and 2^-21 of the exponent; both enter numerator
    and denominator.  Beside bf16 values probabilities come in two pieces, the upper cut off (2^-7), the lower rounded (2^-8): 2^-15 together.
    Beside 8-bit values each, times v_scale_t, is one fp16 number, rounded by 2^-11, or by 2^-25 where the largest of them is at least 2^6: 2^-31 of
    the largest for each stored value.  Values are summed in fp32: n / 16 matrix products and 40 joins one behind the other at most, each good to
    2^-23; factors of running maxima that move take 2^-18.  The result is rounded to bf16, 2^-8."""
    n, Hk, D = k.shape
    qg = q.view(Hk, -1, D)
    s = torch.einsum("kgd,tkd->kgt", qg, k) * scale
    size = torch.einsum("kgd,tkd->kgt", qg.abs(), k.abs()).amax(-1, keepdim=True) * scale
    off = (D + 8) * 2 ** -24 * size + 2 ** -21 * s.abs().amax(-1, keepdim=True) + 2 ** -22
    p = torch.softmax(s, -1)
    ref = torch.einsum("kgt,tkd->kgd", p, v)
    mass = torch.einsum("kgt,tkd->kgd", p, v.abs())
    bound = 2 ** -8 * ref.abs() + mass * ((2 ** -15 if v_scale is None else 2 ** -11) + 2 * off + (n / 16 + 40) * 2 ** -23 + 2 ** -18)
    if v_scale is not None:
        bound += 2 ** -31 * (p * v_scale.t()[:, None]).amax(-1, keepdim=True) * (v.abs() / v_scale[..., None]).sum(0)[:, None]
    return ref.reshape(-1, D), bound.reshape(-1, D)


def scales_of(pages, table, b, n):
    at = torch.arange(n, device="cuda")
    return None if pages.v_scale is None else pages.v_scale[table[b].long()[at // pages.page_size], :, at % pages.page_size].double()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D,page", [(8, 2, 64, 16), (32, 8, 128, 64), (12, 1, 128, 32), (8, 1, 256, 32)])
@pytest.mark.parametrize("n", [1, 10, 40, 1000, 9000])
def test_probabilities_keep_their_bits(dtype, Hq, Hk, D, page, n):
    """probabilities that are nearly alike beside values of alternating signs: the result is far smaller than its terms, so that its own
    rounding hides little"""
    lengths = (n, max(1, n // 3))
    pages, table = filled(2, lengths, Hk, D, page, TYPES[dtype], n)
    sign = 1 - 2 * (torch.arange(page, device="cuda") % 2)
    pages.v.copy_((pages.v.float()[:, :, :1].abs().nan_to_num(1.0) * sign[:, None]).to(pages.v.dtype))
    if pages.v_scale is not None:
        pages.v_scale.copy_(pages.v_scale.nan_to_num(1.0)[:, :, :1].expand_as(pages.v_scale))
    q = draw((2, 1, Hq, D), 5, 0.02)
    out = ops.paged_attention(q, pages, table, ints(*lengths))
    for b, m in enumerate(lengths):
        k, v = stands_for(pages, table, b, m)
        ref, bound = tight_bound(q[b, 0].double(), k, v, D ** -0.5, scales_of(pages, table, b, m))
        far = (out[b, 0].double() - ref).abs()
        assert (far <= bound).all(), (b, m, (far / bound).max().item())


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
@pytest.mark.parametrize("n", [20, 2000])
def test_faint_tokens_beside_one_that_takes_nearly_all(dtype, n):
    """the token with the largest share holds zeros in half of the channels: there the others, 2^-10 to 2^-20 of it, are the result"""
    D = 128
    pages, table = filled(1, (n,), 1, D, 16, TYPES[dtype], 7)
    pages.k.view(torch.uint8).zero_()
    first = table[0, 0].item()
    one = torch.full((D,), 64.0, device="cuda")
    pages.k[first, 0, 5] = one.to(pages.k.dtype)
    pages.k_scale.fill_(1.0 / 64)
    pages.v.view(torch.uint8)[first, 0, 5, : D // 2] = 0
    pages.v_scale.copy_(pages.v_scale.nan_to_num(0.01).clamp(0.005, 0.02))
    for power in (10, 17, 20):
        q = torch.full((1, 1, 4, D), power * 0.6931 * D ** 0.5 / D, device="cuda").bfloat16()       # the first's score: `power` in bits
        out = ops.paged_attention(q, pages, table, ints(n))
        k, v = stands_for(pages, table, 0, n)
        ref, bound = tight_bound(q[0, 0].double(), k, v, D ** -0.5, scales_of(pages, table, 0, n))
        far = (out[0, 0].double() - ref).abs()
        assert (far <= bound).all(), (power, (far / bound).max().item())


@pytest.mark.parametrize("dtype", ["e4m3", "int8"])
def test_scales_as_far_apart_as_fp32_goes(dtype):
    """a row of huge values that has no probability beside rows of tiny ones, and a row that is not a number"""
    pages, table = filled(1, (60,), 1, 128, 16, TYPES[dtype], 9)
    pages.v_scale.fill_(2.0 ** -119)
    far = table[0, 1].item()
    pages.v_scale[far, 0, 3] = 2.0 ** 118
    pages.k.view(torch.uint8).zero_()
    pages.k_scale.fill_(1.0)
    pages.k[far, 0, 3] = torch.full((128,), -100.0, device="cuda").to(pages.k.dtype)
    q = torch.full((1, 1, 4, 128), 4.0, device="cuda").bfloat16()
    check_attention(q, pages, table, (60,), ops.paged_attention(q, pages, table, ints(60)))
    pages.v_scale[far, 0, 3] = float("nan")
    assert ops.paged_attention(q, pages, table, ints(60)).isnan().all()


def test_a_bad_index_does_not_end_the_waits_of_others():
    """a page that does not exist is reported; a flag wait behind it still takes its full time, and its time-out is not overwritten"""
    import time
    from state_space_models_neuron_b200.ops import cuda_ops
    pages, table = filled(1, (40,), 1, 64, 16, torch.bfloat16, 1)
    bad = table.clone()
    bad[0, 1] = -1
    q, flags = draw((1, 1, 1, 64), 2), torch.zeros(64, dtype=torch.int32, device="cuda")
    ops.paged_attention(q, pages, bad, ints(40))
    torch.cuda.synchronize()
    began = time.time()
    cuda_ops._run("ssm_zero1_wait", cuda_ops._P(flags), 0, 2, 5, None, cuda_ops._P(cuda_ops.status_tensor(flags.device)), cuda_ops._st())
    torch.cuda.synchronize()
    assert time.time() - began > 1.0                                   # the limit of a wait is two seconds
    ops.kv_cache_read(pages, bad, ints(40), 40)
    with pytest.raises(RuntimeError, match="status 2 and status 3"):
        cuda_ops.check_status()
    cuda_ops.check_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_traced_calls(dtype):
    """a trace makes the calls again: other tokens, lengths and queries than those that it was made with"""
    pages, table = filled(2, (40, 60), 2, 128, 16, TYPES[dtype], 1)
    pages, table = ops.KVPages(*(None if t is None else t.clone() for t in pages)), table.contiguous()
    copies = [None if t is None else t.clone() for t in pages]
    w = torch.rand(128, device="cuda") + 0.5

    def layer(qkv, n, *held):
        over = ops.KVPages(*held, *[None] * (4 - len(held)))
        q = ops.kv_cache_write(qkv[:, :, 8:10], qkv[:, :, 10:], over, table, n, q=qkv[:, :, :8], q_weight=w, k_weight=w)
        o = ops.paged_attention(q, over, table, n)
        k, v = ops.kv_cache_read(over, table, n, 64)
        return o, k, v

    held, kept = [t for t in pages if t is not None], [t for t in copies if t is not None]
    with torch.no_grad():
        traced = torch.jit.trace(layer, (draw((2, 1, 12, 128), 2), ints(41, 61), *(t.clone() for t in held)), check_trace=False)
        x, n = draw((2, 1, 12, 128), 3), ints(33, 62)
        got, want = traced(x, n, *held), layer(x, n, *kept)
    assert all(same_bits(a, b) for a, b in zip(got, want))              # the second sequence has a token that was never written: NaN
    assert all(same_bits(a, b) for a, b in zip(held, kept))


def test_traced_norms():
    w = torch.rand(128, device="cuda") + 0.5
    cos, sin = ops.rotary_tables(64, 64, 1e4, device="cuda")
    call = lambda q, k, at: ops.qk_norm_rotary(q, k, w, None, 1e-5, cos, sin, at)  # noqa: E731
    x, at = draw((2, 7, 6, 128), 1), torch.arange(14, device="cuda").view(2, 7)
    with torch.no_grad():
        traced = torch.jit.trace(call, (x[:, :, :4], x[:, :, 4:], at), check_trace=False)
        y = draw((2, 7, 6, 128), 2)
        got, want = traced(y[:, :, :4], y[:, :, 4:], at + 3), call(y[:, :, :4], y[:, :, 4:], at + 3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_tangents_are_refused():
    pages, table = filled(1, (40,), 2, 128, 16, torch.bfloat16, 1)
    q = draw((1, 1, 8, 128), 2)
    with torch.autograd.forward_ad.dual_level():
        plain = ops.paged_attention(q, pages, table, ints(40))
        with pytest.raises((NotImplementedError, RuntimeError)):
            ops.paged_attention(torch.autograd.forward_ad.make_dual(q, q), pages, table, ints(40))
    assert torch.equal(plain, ops.paged_attention(q, pages, table, ints(40)))


def spread(n, low, high, empty=()):
    """n lengths between low and high in no order, with some sequences without tokens"""
    out = [low + (i * 7919 + 13) % (high - low + 1) for i in range(n)]
    for i in empty:
        out[i] = -(i % 2)
    return out


SPLITS = [
    # (who takes the work, lengths for rows of up to 64, 128 and more bytes a token and head, query heads, key heads)
    ("item", {64: spread(9, 1, 5000, (0, 4)), 128: spread(9, 1, 5000, (0, 4)), 256: spread(9, 1, 5000, (0, 4))}, 12, 3),
    ("block", {64: spread(40, 2500, 6000, (0, 7, 39)), 128: spread(40, 1300, 4000, (0, 7, 39)), 256: spread(40, 800, 4000, (0, 7, 39))}, 16, 8),
    ("block", {64: spread(120, 3100, 4200, (3,)), 128: spread(120, 1536, 1900, (3,)), 256: spread(120, 768, 1100, (3,))}, 8, 4),
    ("block", {64: spread(70, 4000, 6000), 128: spread(70, 2000, 3000), 256: spread(70, 1000, 1700)}, 70, 5),
    ("warp", {64: spread(100, 1, 900, (0, 50, 99)), 128: spread(100, 1, 500, (0, 50, 99)), 256: spread(100, 1, 300, (0, 50, 99))}, 32, 8),
    ("warp", {64: [1] * 300, 128: [1] * 300, 256: [1] * 300}, 24, 2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("split", range(len(SPLITS)))
def test_every_way_of_sharing_the_work(dtype, D, split):
    """blocks of one item, blocks and warps in equal shares of all items: results, the same bits at every run beside workspaces that
    hold anything, and a graph's replays"""
    from state_space_models_neuron_b200.utils.debug import paged_attention_plan
    by, lengths, Hq, Hk = SPLITS[split]
    row = D * TYPES[dtype].itemsize
    lengths = lengths[min(row, 256)]
    pages, table = filled(len(lengths), lengths, Hk, D, 64, TYPES[dtype], split)
    q, n = draw((len(lengths), 1, Hq, D), 5, 1.5), ints(*lengths)
    plan = paged_attention_plan(q.shape, pages, table.shape[1], lengths)
    assert plan["by"] == by, plan
    first = ops.paged_attention(q, pages, table, n)
    check_attention(q, pages, table, lengths, first)
    for size in (1 << 16, 1 << 20, 1 << 24):
        for _ in range(3):
            junk = torch.full((size,), float("nan"), device="cuda")
            del junk
            assert torch.equal(ops.paged_attention(q, pages, table, n), first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            out = ops.paged_attention(q, pages, table, n)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, first)


@pytest.mark.parametrize("width,spare", [(0, 3), (2, -4)])
def test_tokens_without_any_page_are_reported(width, spare):
    """a table without columns, a pool without pages: tokens are left out, and that is said as for one page that is missing"""
    from state_space_models_neuron_b200.ops import cuda_ops
    pages, table = make_pool(2, width, 2, 16, 128, torch.bfloat16, spare=max(0, spare))
    if spare < 0:
        pages = ops.kv_pages(0, 2, 16, 128, torch.bfloat16, "cuda")
    table = table.view(2, width)
    q = draw((2, 1, 4, 128), 1)
    assert not ops.paged_attention(q, pages, table, ints(0, -3)).any()
    cuda_ops.check_status()
    for lengths in ((0, 5), (5, 5)):
        assert not ops.paged_attention(q, pages, table, ints(*lengths)).any()
        with pytest.raises(RuntimeError, match="status 3"):
            cuda_ops.check_status()
        read = ops.kv_cache_read(pages, table, ints(*lengths), 6)
        assert not read[0].any() and not read[1].any()
        with pytest.raises(RuntimeError, match="status 3"):
            cuda_ops.check_status()
        x = draw((2, 1, 2, 128), 2)
        assert not ops.kv_cache_write(x, x, pages, table, ints(*lengths), q=q)[1].any()
        with pytest.raises(RuntimeError, match="status 3"):
            cuda_ops.check_status()
