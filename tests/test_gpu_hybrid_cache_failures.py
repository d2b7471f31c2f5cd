"""Hybrid models on the GPU behind calls that failed and in inference mode."""
import pytest
import torch

from tests.test_gpu_hybrid_decode import build, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("good", [0, 1, 2])
@torch.no_grad()
def test_a_graph_that_could_not_be_made(good, monkeypatch):
    """the model's head raises in the first or second warm-up step or in the captured one"""
    from state_space_models_neuron_b200.parallel.graph import GraphedDecodeStep
    model, ids = build(), tokens(2, 128)
    cache = model.new_cache(2, 140, page_size=16)
    model.prefill(ids, cache)
    kept = [t.clone() for t in cache.step_state()]
    want = model.step(ids[:, :1], cache)
    for t, k in zip(cache.step_state(), kept):
        t.copy_(k)
    cache.seqlen_offset = 128
    calls, layer = [0], model.backbone.layers[-1]
    plain = layer.step

    def step(*args):
        calls[0] += 1
        if calls[0] > good:
            raise ValueError("no")
        return plain(*args)

    monkeypatch.setattr(layer, "step", step)
    with pytest.raises(ValueError, match="no"):
        GraphedDecodeStep(model, cache, 2)
    monkeypatch.undo()
    assert cache.seqlen_offset == 128 and all(torch.equal(t, k) for t, k in zip(cache.step_state(), kept))
    graph = GraphedDecodeStep(model, cache, 2)
    graph(ids[:, :1])
    assert torch.equal(graph.logits, want)
    cache.torn = True                                                  # what an eager step that failed leaves
    with pytest.raises(RuntimeError, match="reset"):
        graph(ids[:, :1])
    with pytest.raises(RuntimeError, match="reset"):
        GraphedDecodeStep(model, cache, 2)
    assert cache.torn


def test_training_behind_inference_mode():
    """tables and caches first made in inference mode are ordinary tensors to a training step of the same length"""
    from state_space_models_neuron_b200.ops import cuda_ops
    for options in (dict(), dict(qk_norm=False)):
        cuda_ops._ROPE_TABLES.clear()
        cuda_ops._ROPE_VIEWS.clear()
        model, ids = build(**options), tokens(2, 128)
        with torch.inference_mode():
            want = model(input_ids=ids, labels=ids).loss
            model.generate(ids, max_new_tokens=2)
        loss = model(input_ids=ids, labels=ids).loss
        loss.backward()
        assert torch.equal(loss.detach(), want)
