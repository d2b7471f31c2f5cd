"""The bound that the GPU tests put on the attention's probabilities, against models of its arithmetic on the CPU: what the kernel does
stays within it; probabilities in one bf16 piece, or in fp16 without room below the largest, do not."""
import pytest
import torch

from tests.test_gpu_kv_cache_edges import tight_bound


def cut(x):
    """fp32 -> bf16, lower bits cut off"""
    return (x.float().view(torch.int32) & -65536).view(torch.float32)


def attend_bf16(q, k, v, scale, pieces):
    s = torch.einsum("hd,td->ht", q, k) * scale
    e = torch.exp(s - s.amax(-1, keepdim=True)).float()
    top = cut(e)
    p = top.double() + ((e - top).bfloat16().double() if pieces == 2 else 0)
    return (p @ v / e.double().sum(-1, keepdim=True)).bfloat16().double()


def attend_8_bits(q, k, v, scale, v_scale, bits):
    """shares whose largest is in [2^bits, 2^(bits + 1))"""
    s = torch.einsum("hd,td->ht", q, k) * scale
    e = torch.exp(s - s.amax(-1, keepdim=True)).float()
    w = (e.double() * v_scale).float()
    unit = torch.exp2(torch.floor(torch.log2(w.amax(-1, keepdim=True))) - bits)
    return ((w / unit).half().double() @ (v / v_scale[:, None]) * unit.double() / e.double().sum(-1, keepdim=True)).bfloat16().double()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [10, 40])
def test_the_bound_sees_a_missing_piece(D, n):
    g = torch.Generator().manual_seed(n + D)
    q, k = (torch.randn(8, D, generator=g, dtype=torch.float64) * 0.02), torch.randn(n, D, generator=g, dtype=torch.float64)
    v = (1 - 2 * (torch.arange(n) % 2))[:, None] * torch.randint(1, 127, (D,), generator=g).double() * 2.0 ** -7
    ref, bound = tight_bound(q, k[:, None], v[:, None], D ** -0.5)
    for pieces, within in ((2, True), (1, False)):
        far = (attend_bf16(q, k, v, D ** -0.5, pieces) - ref).abs()
        assert bool((far <= bound).all()) is within


@pytest.mark.parametrize("power", [17, 20])
def test_the_bound_sees_faint_shares_that_are_lost(power):
    n, D = 20, 128
    g = torch.Generator().manual_seed(power)
    k, v = torch.zeros(n, D, dtype=torch.float64), torch.randint(-127, 128, (n, D), generator=g).double()
    k[5] = 1
    v[5, : D // 2] = 0
    v_scale = 0.005 + 0.015 * torch.rand(n, generator=g, dtype=torch.float64)
    v = v * v_scale[:, None]
    q = torch.full((4, D), power * 0.6931 * D ** 0.5 / D, dtype=torch.float64)
    ref, bound = tight_bound(q, k[:, None], v[:, None], D ** -0.5, v_scale[:, None])
    for bits, within in ((6, True), (-1, False)):
        far = (attend_8_bits(q, k, v, D ** -0.5, v_scale, bits) - ref).abs()
        assert bool((far <= bound).all()) is within
