"""Paged key-value cache on the GPU where rounding, schedules and failures meet their edges."""
import pytest
import torch

from state_space_models_neuron_b200 import ops
from tests.test_gpu_kv_cache import TYPES, check_attention, draw, filled, ints, make_pool

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
