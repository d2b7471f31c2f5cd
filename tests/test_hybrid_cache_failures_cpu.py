"""Calls over a hybrid cache that fail: what they leave behind gives right results or is refused."""
import pytest
import torch

from tests.test_hybrid_decode_cpu import build, tokens


def logits_of(model, ids, cache, first, last):
    return torch.cat([model.step(ids[:, i:i + 1], cache) for i in range(first, last)], 1)


@pytest.mark.parametrize("prompt", [100, 128])
@torch.no_grad()
def test_steps_after_a_prompt_that_failed(prompt, monkeypatch):
    model, ids = build(), tokens(2, 256)
    full = model(input_ids=ids).logits
    cache = model.new_cache(2, 140, page_size=16)
    if prompt == 128:                                                  # the last layer, behind a Mamba and an attention layer
        monkeypatch.setattr(model.backbone.layers[-1], "forward", lambda *a, **k: (_ for _ in ()).throw(ValueError("no")))
    with pytest.raises(ValueError):                                    # 100: no multiple of the scan's chunk
        model.prefill(ids[:, :prompt], cache)
    monkeypatch.undo()
    assert cache.seqlen_offset == 0 and cache.lengths.tolist() == [0, 0] and not any(t.any() for t in cache.step_state())
    assert (logits_of(model, ids, cache, 0, 8) - full[:, :8]).abs().max() < 1e-4


@torch.no_grad()
def test_a_step_that_failed_between_layers_is_not_continued(monkeypatch):
    model, ids = build(), tokens(2, 256)
    full = model(input_ids=ids).logits
    cache = model.new_cache(2, 140, page_size=16)
    model.prefill(ids[:, :128], cache)
    monkeypatch.setattr(model.backbone.layers[-1], "step", lambda *a, **k: (_ for _ in ()).throw(ValueError("no")))
    with pytest.raises(ValueError, match="no"):
        model.step(ids[:, 128:129], cache)
    monkeypatch.undo()
    with pytest.raises(RuntimeError, match="reset"):
        model.step(ids[:, 128:129], cache)
    with pytest.raises(RuntimeError, match="reset"):
        model(input_ids=ids[:, 128:129], use_cache=True, cache_params=cache)
    cache.reset()
    model.prefill(ids[:, :128], cache)
    assert (logits_of(model, ids, cache, 128, 132) - full[:, 128:132]).abs().max() < 1e-4


@torch.no_grad()
def test_a_first_step_that_failed_does_not_keep_a_prompt_away(monkeypatch):
    model, ids = build(), tokens(2, 256)
    full = model(input_ids=ids).logits
    cache = model.new_cache(2, 140, page_size=16)
    monkeypatch.setattr(model.backbone.layers[-1], "step", lambda *a, **k: (_ for _ in ()).throw(ValueError("no")))
    with pytest.raises(ValueError, match="no"):
        model.step(ids[:, :1], cache)
    monkeypatch.undo()
    model.prefill(ids[:, :128], cache)
    assert (logits_of(model, ids, cache, 128, 132) - full[:, 128:132]).abs().max() < 1e-4


@torch.no_grad()
def test_calls_that_do_not_fit_leave_the_cache_as_it_was():
    model, ids = build(), tokens(3, 256)
    full = model(input_ids=ids[:2]).logits
    cache = model.new_cache(2, 140, page_size=16)
    for wrong in (lambda: model.prefill(ids[:, :128], cache), lambda: model.step(ids[:, :1], cache), lambda: model.step(ids[:2, :2], cache)):
        with pytest.raises(ValueError):
            wrong()
        assert cache.seqlen_offset == 0 and cache.lengths.tolist() == [0, 0]
    model.prefill(ids[:2, :128], cache)
    for wrong in (lambda: model.step(ids[:, 128:129], cache), lambda: model.step(ids[:2, 128:130], cache),
                  lambda: model(input_ids=ids[:2, 128:130], use_cache=True, cache_params=cache)):
        with pytest.raises(ValueError):
            wrong()
    assert (logits_of(model, ids[:2], cache, 128, 140) - full[:, 128:140]).abs().max() < 1e-4
    with pytest.raises(ValueError, match="room for 140"):
        model.step(ids[:2, :1], cache)


def test_caches_made_in_inference_mode_and_used_outside():
    model, ids = build(), tokens(2, 256)
    with torch.inference_mode():
        full = model(input_ids=ids).logits
        _, cache = model.prefill(ids[:, :128])
        first = model.step(ids[:, 128:129], cache)
    with torch.no_grad():
        got = torch.cat([first] + [model.step(ids[:, i:i + 1], cache) for i in range(129, 136)], 1)
    assert (got - full[:, 128:136]).abs().max() < 1e-4
    cache.reset()
    assert cache.lengths.tolist() == [0, 0]
