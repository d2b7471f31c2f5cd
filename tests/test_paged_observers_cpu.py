"""Operators over pages under tracing and forward-mode differentiation, with a stand-in that fills its results through their
addresses, as the kernels do."""
import contextlib

import pytest
import torch

from state_space_models_neuron_b200.ops import KVPages, cuda_ops


@pytest.fixture(autouse=True)
def _cpu(monkeypatch):
    """the current device is the CPU's number, and no other is made current"""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())


@cuda_ops._over_pages(1)
def read(x, pages, more, none, factor):
    out = torch.empty_like(x)
    out.numpy()[:] = factor * (x.detach().numpy() + pages.k.numpy() + more.numpy())
    return out


@cuda_ops._over_pages(0)
def write(pages, x):
    pages.k.numpy()[:] = x.numpy()


def test_traces_make_the_call():
    def both(x, k, more):
        pages = KVPages(k, k)
        write(pages, x * 2)
        return read(x, pages, more, None, 3.0) + 1

    with torch.no_grad():
        traced = torch.jit.trace(both, (torch.ones(4), torch.zeros(4), torch.zeros(4)), check_trace=False)
        k = torch.zeros(4)
        out = traced(torch.full((4,), 5.0), k, torch.ones(4))
    assert torch.equal(out, torch.full((4,), 3 * (5.0 + 10.0 + 1.0) + 1)) and torch.equal(k, torch.full((4,), 10.0))


def test_plain_calls_are_plain(monkeypatch):
    monkeypatch.setattr(cuda_ops._OverPages, "apply", None)
    k = torch.zeros(4)
    assert write(KVPages(k, k), torch.ones(4)) is None
    assert torch.equal(read(torch.ones(4), KVPages(k, k), k, None, 2.0), torch.full((4,), 6.0))       # k is `more` as well


def test_tangents_are_refused():
    k = torch.zeros(4)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        assert torch.equal(read(torch.ones(4), KVPages(k, k), k, None, 2.0), torch.full((4,), 2.0))
        dual = torch.autograd.forward_ad.make_dual(torch.ones(4), torch.ones(4))
        with pytest.raises((NotImplementedError, RuntimeError)):
            read(dual, KVPages(k, k), k, None, 2.0)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda t: read(t, KVPages(k, k), k, None, 2.0))(torch.ones(2, 4))


def test_nothing_is_differentiable():
    k = torch.zeros(4)
    x = torch.ones(4, requires_grad=True)
    with torch.autograd.forward_ad.dual_level():
        out = read(x, KVPages(k, k), k, None, 2.0)
    assert not out.requires_grad and torch.equal(out, torch.full((4,), 2.0))


def test_calls_inside_a_transform_of_something_else():
    """constants to the function that is differentiated, as they are outside of it"""
    k = torch.zeros(4)

    def loss(w):
        write(KVPages(k, k), torch.full((4,), 2.0))
        return (w * read(torch.ones(4), KVPages(k, k), torch.zeros(4), None, 2.0)).sum()

    assert torch.equal(torch.func.grad(loss)(torch.ones(4)), torch.full((4,), 6.0)) and torch.equal(k, torch.full((4,), 2.0))
