"""Hybrid model with norms of queries and keys and a paged cache on the GPU: training, prompts, decoding, graphs."""
import pytest
import torch

from state_space_models_neuron_b200 import ops
from state_space_models_neuron_b200.models import Mamba2HybridConfig, Mamba2HybridForCausalLM
from state_space_models_neuron_b200.parallel import state as ps

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    from state_space_models_neuron_b200.ops import cuda_ops
    torch.cuda.synchronize()
    cuda_ops.check_status()


def build(**options):
    ps.initialize_model_parallel(1)
    kw = dict(num_heads=8, head_dim=64, vocab_size=512, hidden_size=256, state_size=128, num_hidden_layers=5, n_groups=1,
              attn_num_heads=8, attn_head_dim=128, attn_key_value_heads=2, mlp_hidden_size=512, hybrid_override_pattern="M*-M*",
              initializer_range=0.05, dtype=torch.bfloat16, qk_norm=True, rotary_emb_dim=64)
    torch.manual_seed(0)
    model = Mamba2HybridForCausalLM(Mamba2HybridConfig(**{**kw, **options}), device="cuda").to(torch.bfloat16).eval()
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "q_norm" in n or "k_norm" in n:
                p.copy_(torch.rand(p.shape, generator=torch.Generator().manual_seed(len(n))) + 0.5)
    return model


def tokens(B, L):
    return torch.randint(0, 512, (B, L), generator=torch.Generator().manual_seed(B + L)).cuda()


def near(a, b, ratio):
    """the bounds of the decode check of `mamba2_inference.py`: bf16 passes in another order, mean error as a share of the spread"""
    err, std = (a - b).abs(), b.std()
    assert err.mean() <= ratio * std and err.max() <= std * max(1.0, 10 * ratio), (err.mean() / std, err.max() / std)


@pytest.mark.parametrize("options", [dict(), dict(qk_norm=False), dict(rotary_emb_dim=None), dict(qk_norm=False, rotary_emb_dim=None)])
@pytest.mark.parametrize("kv,ratio", [(None, 3e-2), (torch.int8, 4e-2), (torch.float8_e4m3fn, 0.1)])
@torch.no_grad()
def test_decoding_is_the_forward_pass(options, kv, ratio):
    model = build(**options)
    ids = tokens(3, 256)
    full = model(input_ids=ids).logits
    cache = model.new_cache(3, 256, kv_dtype=kv, page_size=32)
    first, _ = model.prefill(ids[:, :128], cache)
    near(first[:, 0], full[:, 127], 3e-2)
    got = torch.cat([model.step(ids[:, i:i + 1], cache) for i in range(128, 256)], 1)
    near(got, full[:, 128:], ratio)


@torch.no_grad()
def test_the_cache_holds_the_keys_and_values_of_the_prompt():
    model = build()
    ids = tokens(2, 128)
    held = {}
    layer = model.backbone.layers[1].layer
    plain = layer._queries_keys_values

    def keep(x):
        held["qkv"] = plain(x)
        return held["qkv"]

    layer._queries_keys_values = keep
    _, cache = model.prefill(ids)
    q, k, v = held["qkv"]
    cos, sin = ops.rotary_tables(128, 64, layer.rope_theta, device=q.device)
    _, want = ops.qk_norm_rotary(q, k, layer.q_norm.weight, layer.k_norm.weight, layer.norm_eps, cos, sin)
    got = cache.keys_values(1)
    assert torch.equal(got[0], want) and torch.equal(got[1], v)


@pytest.mark.parametrize("kv", [None, torch.int8, torch.float8_e4m3fn])
@torch.no_grad()
def test_graph_gives_the_tokens_of_eager_steps(kv):
    from state_space_models_neuron_b200.parallel.graph import GraphedDecodeStep
    model = build()
    ids = tokens(5, 128)
    runs = []
    for graphed in (False, True):
        cache = model.new_cache(5, 140, kv_dtype=kv, page_size=16)
        logits, _ = model.prefill(ids, cache)
        tok = logits[:, -1].argmax(-1, keepdim=True)
        step = GraphedDecodeStep(model, cache, 5) if graphed else None
        assert cache.seqlen_offset == 128 and cache.lengths.tolist() == [128] * 5
        out = []
        for _ in range(12):
            if graphed:
                tok = step(tok).clone()
                out.append((step.logits.clone(), tok))
            else:
                logits = model.step(tok, cache)
                tok = logits[:, -1].argmax(-1, keepdim=True)
                out.append((logits, tok))
        with pytest.raises(ValueError, match="room for 140"):
            step(tok) if graphed else model.step(tok, cache)
        runs.append(out)
    for (a, s), (b, t) in zip(*runs):
        assert torch.equal(a, b) and torch.equal(s, t)


@torch.no_grad()
def test_a_graph_of_a_cache_with_room_for_one_token():
    from state_space_models_neuron_b200.parallel.graph import GraphedDecodeStep
    model = build()
    ids = tokens(2, 128)
    cache = model.new_cache(2, 129, page_size=16)
    model.prefill(ids, cache)
    step = GraphedDecodeStep(model, cache, 2)
    step(ids[:, :1])
    assert cache.lengths.tolist() == [129, 129]


@torch.no_grad()
def test_generate():
    model = build()
    out = model.generate(tokens(2, 150), max_new_tokens=7, do_sample=False)
    assert out.shape == (2, 157) and torch.equal(out[:, :150], tokens(2, 150))


def test_training_gradients_are_those_of_the_fp32_model():
    """bf16 kernels against the same weights and the operators' plain forms in fp32 on the CPU, as far as bf16 activations agree"""
    model = build().train()
    ids = tokens(2, 128)
    loss = model(input_ids=ids, labels=ids).loss
    loss.backward()
    sd = {k: v.float().cpu() for k, v in model.state_dict().items()}
    plain = Mamba2HybridForCausalLM(model.config).float()
    plain.load_state_dict(sd)
    ref = plain(input_ids=ids.cpu(), labels=ids.cpu()).loss
    ref.backward()
    assert abs(loss.item() - ref.item()) < 2e-2 * ref.item()
    theirs = dict(plain.named_parameters())
    for n, p in model.named_parameters():
        if "q_norm" in n or "k_norm" in n or "q_proj" in n or "k_proj" in n:
            a, b = p.grad.float().cpu().flatten(), theirs[n].grad.flatten()
            assert torch.dot(a, b) > 0.95 * a.norm() * b.norm(), n


def test_training_step_in_a_graph():
    from state_space_models_neuron_b200 import parallel as nxd
    from state_space_models_neuron_b200.parallel.graph import GraphedTrainStep
    ids = tokens(2, 128)

    weights = build().state_dict()                                 # every construction draws others

    def start():
        model = build().train()
        model.load_state_dict(weights)
        cfg = nxd.parallel_config(1, {"zero_one_enabled": True})
        return model, nxd.initialize_parallel_optimizer(cfg, nxd.AdamW_FP32OptimParams, [{"params": list(model.parameters())}], lr=1e-3)

    model, opt = start()
    losses = []
    for _ in range(4):
        opt.zero_grad()
        loss = model(input_ids=ids, labels=ids, return_logits=False).loss
        loss.backward()
        opt.step()
        losses.append(loss.item())
    before = [p.detach().clone() for n, p in model.named_parameters() if "q_norm" in n or "k_norm" in n]
    assert all(not torch.equal(p, torch.ones_like(p)) for p in before)
    model, opt = start()
    step = GraphedTrainStep(model, opt, {"input_ids": ids, "labels": ids}, warmup=2)
    graphed = [step({"input_ids": ids, "labels": ids}).item() for _ in range(2)]
    # the same kernels in the same order; sums over tokens by atomics (embedding, scan) may differ in their last bits
    for a, b in zip(losses[2:], graphed):
        assert abs(a - b) < 2e-2 * a
