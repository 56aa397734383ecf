"""The few-token experts inside a model: the same answers with the option and without, by two launches a layer, at every width."""

import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks
from tiny_llm_b200 import greedy_generate_ids
from tiny_llm_b200.mlp import FewTokenExperts, MixtureOfExperts, TopKRouter
from tiny_llm_b200.models import model_class
from tiny_llm_b200.synthetic import synthetic_voluzen, voluzen_config

from tests import test_gpu_voluzen as V
from tests.test_gpu_moe_few import make

DEV = "cuda"
pytestmark = pytest.mark.gpu

CONFIGS = {
    "whole": dict(pattern="CSM", experts=8, top=2, expert_ff=64),
    "awkward": dict(pattern="CSMC", width=100, heads=3, experts=5, top=2, expert_ff=20),  # rows that are no whole 16-byte pieces
}


@pytest.mark.parametrize("name", CONFIGS)
def test_a_model_answers_as_without(name, monkeypatch):
    config = voluzen_config(**CONFIGS[name])
    tensors = V.decisive_routers(synthetic_voluzen(config, seed=5))
    plain, few = (model_class("Voluzen")(config, tensors, few_token_experts=option) for option in (False, True))
    layers = [layer.mlp for layer in few.layers if isinstance(layer.mlp, MixtureOfExperts)]
    assert layers and all(m.few is not None for m in layers)
    calls = []
    inner = FewTokenExperts.__call__
    monkeypatch.setattr(FewTokenExperts, "__call__", lambda self, h, wide=False: (calls.append(h.shape[0]), inner(self, h, wide))[1])
    prompt = [3, 17, 5, 99, 42, 7]
    logits = [model(torch.tensor([prompt], device=DEV), 0, model.create_kv_cache())[0].double().cpu() for model in (plain, few)]
    assert calls == [len(prompt)] * len(layers)
    assert V.rows_match(logits[1], logits[0], torch.bfloat16)
    del calls[:]
    steps = 6
    got = [greedy_generate_ids(model, prompt, steps) for model in (plain, few)]
    assert got[0] == got[1] and len(got[0]) >= steps
    # the prompt; of the steps of one token the first, and the one that is captured (the others are its replays)
    assert calls.count(len(prompt)) == len(layers) and calls.count(1) == 2 * len(layers) and few.graph_replays >= steps - 2


@pytest.mark.parametrize("D", [64, 100])
def test_two_launches_a_layer(D):
    h, router, wg, wu, wd = make(3, D, 64, 8, False)
    layer = MixtureOfExperts(TopKRouter(router, None, 2), wg, wu, wd, "silu")
    counts = []
    for use in (False, True):
        if use:
            layer.use_few_tokens()
        layer(h)
        before = blocks.launch_count()
        y = layer(h)
        counts.append(blocks.launch_count() - before)
        assert y.is_contiguous() and y.shape == (3, D) and y.dtype == torch.float32
    assert counts[1] == 2 < counts[0]


def test_steps_of_more_tokens_keep_to_the_chain():
    most = MixtureOfExperts.FEW_TOKENS
    h, router, wg, wu, wd = make(most + 1, 64, 64, 8, False)
    chain = MixtureOfExperts(TopKRouter(router, None, 2), wg, wu, wd, "silu")
    few = MixtureOfExperts(chain.router, wg, wu, wd, "silu").use_few_tokens()
    assert torch.equal(few(h), chain(h))
    assert torch.equal(few(h[:most]), few.few(h[:most], wide=True)) and not torch.equal(few(h[:most]), chain(h[:most]))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T", [1, 5, 40])
def test_outputs_of_odd_widths_are_whole(T, eight):
    h, router, wg, wu, wd = make(T, 100, 50, 6, eight)
    layer = FewTokenExperts(TopKRouter(router, None, 2), wg, wu, wd, "silu")
    assert all(layer(h, wide=wide).is_contiguous() for wide in (False, True))
