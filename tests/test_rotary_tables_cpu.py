"""Tables of the rotary embedding as the GPU path keeps them (built here on the CPU)."""
import pytest
import torch

from state_space_models_neuron_b200.ops import cuda_ops, oracle


@pytest.fixture(autouse=True)
def _empty(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_ROPE_TABLES", {})
    monkeypatch.setattr(cuda_ops, "_ROPE_VIEWS", {}, raising=False)


@pytest.mark.parametrize("L,dim,offset", [(1, 64, 0), (2, 8, 0), (100, 128, 0), (129, 64, 7), (5, 6, 1), (3, 64, 4096), (4, 64, -2)])
def test_rows_are_those_of_the_definition(L, dim, offset):
    got = cuda_ops.rotary_tables(L, dim, 1e4, "cpu", offset)
    for a, b in zip(got, oracle.rotary_tables(L, dim, 1e4, offset=offset)):
        assert torch.equal(a, b) and a.is_contiguous() and a.data_ptr() % 16 == 0


def test_lengths_share_tables():
    """as `generate` asks: every sum of prompt and new tokens is another length"""
    first = cuda_ops.rotary_tables(130, 64, 1e4, "cpu")
    assert cuda_ops.rotary_tables(130, 64, 1e4, "cpu")[0] is first[0]
    for n in range(1, 2001):
        assert cuda_ops.rotary_tables(n, 64, 1e4, "cpu")[0].shape == (n, 32)
    held = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for pair in cuda_ops._ROPE_TABLES.values() for t in pair}
    held.update({t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for pair in cuda_ops._ROPE_VIEWS.values() for t in pair})
    assert sum(held.values()) <= 2 * 2 * 2048 * 32 * 4                  # powers of two up to 2048 positions, cosines and sines
    assert len(cuda_ops._ROPE_VIEWS) <= 256


def test_tables_first_made_in_inference_mode():
    with torch.inference_mode():
        cuda_ops.rotary_tables(16, 8, 1e4, "cpu")
    x = torch.ones(16, 4, requires_grad=True)
    cos, sin = cuda_ops.rotary_tables(16, 8, 1e4, "cpu")
    (x * cos + x * sin).sum().backward()                               # saves the tables
    assert torch.equal(x.grad, cos + sin)
    cos, _ = cuda_ops.rotary_tables(12, 8, 1e4, "cpu")
    (x[:12] * cos).sum().backward()
