"""The rule by which the attention over pages shares its work, as the library applies it (host only, 148 SMs assumed)."""
import pytest
import torch

from state_space_models_neuron_b200 import ops
from state_space_models_neuron_b200.utils.debug import paged_attention_plan
from tests.test_gpu_kv_cache_edges import SPLITS, TYPES


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("split", range(len(SPLITS)))
def test_the_cases_of_the_gpu_tests_reach_what_they_name(dtype, D, split):
    by, lengths, Hq, Hk = SPLITS[split]
    lengths = lengths[min(D * TYPES[dtype].itemsize, 256)]
    pages = ops.kv_pages(1, Hk, 64, D, TYPES[dtype])
    plan = paged_attention_plan((len(lengths), 1, Hq, D), pages, -(-max(lengths) // 64), lengths)
    assert plan["by"] == by, plan
    assert by == "item" or plan["share"] * plan["workers"] >= plan["steps"]
    assert {s[0] for s in SPLITS} == {"item", "block", "warp"}


def test_lengths_behind_the_table_and_below_zero():
    pages = ops.kv_pages(1, 2, 16, 128, torch.bfloat16)
    plan = lambda *n: paged_attention_plan((len(n), 1, 8, 128), pages, 4, n)  # noqa: E731
    assert plan(10 ** 9, -5)["steps"] == plan(64, 0)["steps"] == 8
    with pytest.raises(ValueError):
        paged_attention_plan((1, 1, 7, 128), pages, 4, [1])
