"""Hybrid model with norms of queries and keys and with a key-value cache on the CPU: decoding against the full forward pass, caches,
gradients, tensor parallelism on two gloo ranks, checkpoints, the command."""
import os
import tempfile

import pytest
import torch

from state_space_models_neuron_b200.models import Mamba2HybridCache, Mamba2HybridConfig, Mamba2HybridForCausalLM
from state_space_models_neuron_b200.parallel import state as ps
from tests.dist_utils import run_ranks


def config(sp=False, **options):
    kw = dict(num_heads=4, head_dim=32, vocab_size=256, hidden_size=64, state_size=32, num_hidden_layers=4, n_groups=2,
              tie_word_embeddings=True, initializer_range=0.05, sequence_parallel_enabled=sp, dtype=torch.float32, attn_num_heads=4,
              attn_head_dim=16, attn_key_value_heads=2, mlp_hidden_size=128, hybrid_override_pattern="M*-*", residual_in_fp32=False,
              qk_norm=True, rotary_emb_dim=8)
    return Mamba2HybridConfig(**{**kw, **options})


def build(**options):
    ps.initialize_model_parallel(1)
    torch.manual_seed(0)
    model = Mamba2HybridForCausalLM(config(**options)).eval()
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "q_norm" in n or "k_norm" in n:
                p.copy_(torch.rand_like(p) + 0.5)
    return model


def tokens(B, L, seed=1):
    return torch.randint(0, 256, (B, L), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("options", [dict(), dict(qk_norm=False), dict(qk_norm=False, rotary_emb_dim=None), dict(rotary_emb_dim=None),
                                     dict(qkv_linear=True)])
@torch.no_grad()
def test_steps_are_the_forward_pass(options):
    """fp32 with fp32 pages: the two sum in other orders only; 1e-4 of logits with a standard deviation near 1 is 800 roundings"""
    model = build(**options)
    ids = tokens(2, 256)
    full = model(input_ids=ids).logits
    for start in (0, 128):
        cache = model.new_cache(2, 140, page_size=16)
        outs = []
        if start:
            last, same = model.prefill(ids[:, :start], cache)
            assert same is cache
            outs.append(last)
        outs += [model.step(ids[:, i:i + 1], cache) for i in range(start, 140)]
        got = torch.cat(outs, 1)
        assert (got - full[:, max(0, start - 1):140]).abs().max() < 1e-4
        assert cache.seqlen_offset == 140 and cache.lengths.tolist() == [140, 140]
        k, v = cache.keys_values(1, torch.float32)
        assert k.shape == (2, 140, 2, 16) and k[:, -1].any() and v[:, -1].any()
        with pytest.raises(ValueError, match="room for 140"):
            model.step(ids[:, :1], cache)
        cache.reset()
        again = model.step(ids[:, :1], cache)
        assert (again[:, 0] - full[:, 0]).abs().max() < 1e-4


@pytest.mark.parametrize("dtype,most", [(torch.bfloat16, 0.05), (torch.int8, 0.1), (torch.float8_e4m3fn, 0.5)])
@torch.no_grad()
def test_narrow_pages(dtype, most):
    """keys and values are off by at most half a step, 2^-8, 1/254 of a row's largest and 2^-4: logits by that times a small factor"""
    model = build()
    ids = tokens(2, 128)
    full = model(input_ids=ids).logits
    cache = model.new_cache(2, 32, kv_dtype=dtype, page_size=16)
    got = torch.cat([model.step(ids[:, i:i + 1], cache) for i in range(32)], 1)
    assert (got - full[:, :32]).abs().max() < most * full.std()


@torch.no_grad()
def test_use_cache_in_the_forward_pass_and_generate():
    model = build()
    ids = tokens(2, 256)
    full = model(input_ids=ids).logits
    out = model(input_ids=ids[:, :128], use_cache=True)
    assert out.cache_params.max_length == 8192 and (out.logits - full[:, :128]).abs().max() < 1e-4
    out = model(input_ids=ids[:, 128:129], use_cache=True, cache_params=out.cache_params)
    assert (out.logits[:, 0] - full[:, 128]).abs().max() < 1e-4
    again = model.new_cache(2, 256)
    with pytest.raises(ValueError, match="multiple of"):
        model.prefill(ids[:, :100], again)                         # leaves an empty cache behind
    assert (model.prefill(ids[:, :128], again)[0][:, 0] - full[:, 127]).abs().max() < 1e-4 and again.lengths.tolist() == [128, 128]
    assert (model.step(ids[:, 128:129], again)[:, 0] - full[:, 128]).abs().max() < 1e-4
    with pytest.raises(ValueError, match="empty cache"):
        model(input_ids=ids[:, :128], use_cache=True, cache_params=out.cache_params)
    new = model.generate(ids[:, :130], max_new_tokens=6, do_sample=False)
    assert new.shape == (2, 136)
    for i in range(130, 136):
        padded = torch.cat([new[:, :i], torch.zeros(2, 256 - i, dtype=torch.long)], 1)
        logits = model(input_ids=padded).logits[:, i - 1]
        best = logits.max(-1).values
        # the chosen token is the best one, or as good within the two passes' roundings
        assert (logits.gather(1, new[:, i:i + 1])[:, 0] >= best - 1e-4).all()


def test_training_gradients_against_differences():
    """The loss along its gradient in the norms' weights.  An fp32 loss near 6 is known to 2^-22 (2.4e-7), two of them over a step of
    2 h = 0.1 give the slope to 5e-6, and halving h shows what the curvature adds."""
    model = build()
    params = [p for n, p in model.named_parameters() if "q_norm" in n or "k_norm" in n]
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "q_norm" in n or "k_norm" in n or "v_proj" in n or "o_proj" in n:
                p.mul_(4.0)                                        # sharp scores, whose gradients are not lost in the loss
    ids = tokens(4, 128)
    model(input_ids=ids, labels=ids).loss.backward()
    grads = [p.grad.clone() for p in params]
    norm = torch.sqrt(sum(g.square().sum() for g in grads)).item()
    start = [p.detach().clone() for p in params]

    def slope(h):
        sides = []
        with torch.no_grad():
            for sign in (h, -h):
                for p, q, g in zip(params, start, grads):
                    p.copy_(q + sign * g / norm)
                sides.append(model(input_ids=ids, labels=ids).loss.item())
        return (sides[0] - sides[1]) / (2 * h)

    wide, near = slope(0.1), slope(0.05)
    assert norm > 1e-3 and abs(near - norm) <= abs(wide - near) + 2 * 5e-6


def _single(rank, world, path):
    from state_space_models_neuron_b200 import parallel as nxd
    ps.initialize_model_parallel(1)
    cfg = nxd.parallel_config(1, {"zero_one_enabled": False}, device="cpu", init_seed=7)
    model = nxd.initialize_parallel_model(cfg, lambda: Mamba2HybridForCausalLM(config()))
    opt = nxd.initialize_parallel_optimizer(cfg, nxd.AdamW_FP32OptimParams, [{"params": list(model.parameters())}], lr=1e-2)
    ids = tokens(4, 128, 3)
    losses = []
    for _ in range(3):
        opt.zero_grad()
        loss = model(input_ids=ids, labels=ids).loss
        loss.backward()
        opt.step()
        losses.append(loss.item())
    sd = {k: v.clone() for k, v in model.state_dict().items()}
    model.eval()
    with torch.no_grad():
        cache = model.new_cache(2, 140, page_size=16)
        logits = [model.prefill(ids[:2], cache)[0]] + [model.step(ids[2:, i:i + 1], cache) for i in range(8)]
    torch.save((losses, sd, torch.cat(logits, 1)), path)


def _pair(rank, world, path, sp):
    from state_space_models_neuron_b200 import parallel as nxd
    from state_space_models_neuron_b200.parallel.layout import merge_state_dicts, shard_state_dict
    losses, sd, logits = torch.load(path, weights_only=False)
    ps.initialize_model_parallel(world)
    cfg = nxd.parallel_config(world, {"zero_one_enabled": False}, sequence_parallel=sp, device="cpu", init_seed=7)
    model = nxd.initialize_parallel_model(cfg, lambda: Mamba2HybridForCausalLM(config(sp)))
    opt = nxd.initialize_parallel_optimizer(cfg, nxd.AdamW_FP32OptimParams, [{"params": list(model.parameters())}], lr=1e-2)
    ids = tokens(4, 128, 3)
    for want in losses:
        opt.zero_grad()
        loss = model(input_ids=ids, labels=ids).loss
        loss.backward()
        opt.step()
        assert abs(loss.item() - want) < 2e-4
    mine = {k: v.clone() for k, v in model.state_dict().items()}
    shards = [None] * world
    torch.distributed.all_gather_object(shards, mine)
    merged = merge_state_dicts(shards, config())
    for k, v in sd.items():
        assert torch.allclose(merged[k], v, atol=2e-4, rtol=1e-3), (k, (merged[k] - v).abs().max())
    if sp:
        return
    model.load_state_dict(shard_state_dict(sd, config(), world, rank), strict=False)
    model.eval()
    with torch.no_grad():
        cache = model.new_cache(2, 140, page_size=16)
        assert cache.pages[1].k.shape[1] == 1                       # one of the two key heads
        got = [model.prefill(ids[:2], cache)[0]] + [model.step(ids[2:, i:i + 1], cache) for i in range(8)]
    per = 256 // world
    assert torch.allclose(torch.cat(got, 1), logits[..., rank * per:(rank + 1) * per], atol=3e-4, rtol=1e-3)


@pytest.fixture(scope="module")
def single_run():
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "single.pt")
        run_ranks(_single, 1, path)
        yield path


@pytest.mark.parametrize("sp", [False, True])
def test_two_ranks_train_and_decode_as_one(single_run, sp):
    run_ranks(_pair, 2, single_run, sp)


def test_checkpoint_keeps_the_norms():
    model = build()
    with tempfile.TemporaryDirectory() as d:
        model.save_pretrained(d)
        back = Mamba2HybridForCausalLM.from_pretrained(d)
    assert back.config.qk_norm and back.config.rotary_emb_dim == 8
    for (n, a), (m, b) in zip(sorted(model.state_dict().items()), sorted(back.state_dict().items())):
        assert n == m and torch.equal(a, b)
    plain = Mamba2HybridForCausalLM(config(qk_norm=False))
    assert not any("q_norm" in n or "k_norm" in n for n in plain.state_dict())


def test_cache_layout():
    ps.initialize_model_parallel(1)
    cache = Mamba2HybridCache(config(), 3, 100, dtype=torch.float32, kv_dtype=torch.int8, page_size=32)
    assert sorted(cache.pages) == [1, 3] and sorted(cache.conv_states) == [0]
    assert cache.pages[1].k.shape == (12, 2, 32, 16) and cache.pages[1].k_scale.shape == (12, 2, 32)
    assert sorted(cache.block_table.flatten().tolist()) == list(range(12))


def test_command(capsys):
    import mamba2_inference
    argv = ["--model", "Mamba2Hybrid800M", "--vocab_size", "64", "--dtype", "float32", "--batch", "1", "--seq_len", "128", "--device", "cpu",
            "--qk_norm", "--rotary_emb_dim", "32", "--page_size", "16"]
    from state_space_models_neuron_b200.models import predefined_configs as pc
    sizes = pc.CONFIGS_KWARGS["Mamba2Hybrid800M"]
    pc.CONFIGS_KWARGS["Mamba2Hybrid800M"] = pc.ConfParams(64, 4, head_dim=32)
    try:
        with pytest.raises(SystemExit) as done:
            mamba2_inference.main(argv)
        assert done.value.code == 0
        mamba2_inference.main(argv + ["--mode", "bench", "--decode_tokens", "2", "--warmup", "1", "--kv_cache_dtype", "int8"])
    finally:
        pc.CONFIGS_KWARGS["Mamba2Hybrid800M"] = sizes
    assert '"metric": "decode tokens/s"' in capsys.readouterr().out
