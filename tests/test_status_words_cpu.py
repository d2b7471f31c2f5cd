"""Status words of the native kernels: what the host makes of them (tensors of the CPU stand in for a device's)."""
import pytest
import torch

from state_space_models_neuron_b200.ops import cuda_ops


@pytest.mark.parametrize("words,said", [((1, 0), "status 1 on"), ((2, 0), "status 2 on"), ((0, 3), "status 3 on"), ((2, 3), "status 2 and status 3 on")])
def test_both_words_are_read_and_cleared(monkeypatch, words, said):
    t = torch.tensor(words, dtype=torch.int32)
    monkeypatch.setattr(cuda_ops, "_status", {"a device": torch.zeros(2, dtype=torch.int32), "another": t})
    with pytest.raises(RuntimeError, match=said):
        cuda_ops.check_status()
    assert not t.any()
    cuda_ops.check_status()


def test_a_device_has_two_words(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_status", {})
    t = cuda_ops.status_tensor("cpu")
    assert t.shape == (2,) and not t.any() and cuda_ops.status_tensor("cpu") is t


def test_words_made_in_inference_mode_are_cleared_outside(monkeypatch):
    monkeypatch.setattr(cuda_ops, "_status", {})
    with torch.inference_mode():
        cuda_ops.status_tensor("cpu")[1] = 3
    with pytest.raises(RuntimeError, match="status 3"):
        cuda_ops.check_status()
    cuda_ops.check_status()
