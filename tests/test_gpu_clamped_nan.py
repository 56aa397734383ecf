"""A NaN passes the clamped activation: its bounds are comparisons, and one that answers with the bound would make a number of it.

Every kernel that has the activation: the 8-bit feed-forward in its forms by rows, the experts for few tokens, and the feed-forward and the experts of 16 and 32
bits.  A NaN may come by the gate or by the other half, from a token or from a matrix."""

import pytest
import torch

from tiny_llm_b200.fp8 import Fp8Weights
from tiny_llm_b200.mlp import FewTokenExperts, Fp8GatedMLP, GatedMLP, MixtureOfExperts, TopKRouter

DEV = "cuda"
LIMIT, SLOPE = 1.2, 1.7
pytestmark = pytest.mark.gpu


def rand(seed, *shape, std=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std


def fp8(w):
    q = Fp8Weights.from_tensor(w)
    return Fp8Weights(q.values[..., : w.shape[-1]].to(DEV), q.scales.to(DEV))


def spoil(w, *at):
    """``w`` with a NaN at one entry."""
    if isinstance(w, Fp8Weights):
        values = w.values.clone()
        values.view(torch.uint8)[at] = 0x7F
        return Fp8Weights(values[..., : w.shape[-1]], w.scales)
    w = w.clone()
    w[at] = float("nan")
    return w


@pytest.mark.parametrize("rows", [1, 4, 5, 30, 150, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_8_bit_feed_forward(rows, dtype):
    D, ff = 200, 333
    gate, up, down = fp8(rand(1, ff, D, std=D**-0.5)), fp8(rand(2, ff, D, std=D**-0.5)), fp8(rand(3, D, ff, std=ff**-0.5))
    layer = Fp8GatedMLP(gate, up, down, "clamped_swish", LIMIT, SLOPE)
    x = rand(rows, rows, D).to(dtype).to(DEV)
    want = layer(x)
    assert torch.isfinite(want).all()
    for value in (float("inf"), float("-inf"), float("nan")):
        for row in sorted({0, rows - 1}):
            y = x.clone()
            y[row, 77] = value
            got = layer(y)
            assert torch.isnan(got[row]).all()
            others = torch.arange(rows, device=DEV) != row
            assert torch.equal(got[others], want[others])
    # an inner number that is none takes its run of a row along, and the run every output
    for bad in ((spoil(gate, 3, 5), up), (gate, spoil(up, 300, 199))):
        assert torch.isnan(Fp8GatedMLP(*bad, down, "clamped_swish", LIMIT, SLOPE)(x)).all()


@pytest.mark.parametrize("T", [1, 6, 30])
@pytest.mark.parametrize("eight", [False, True])
def test_experts_for_few_tokens(T, eight):
    D, ff, E, top = 136, 90, 8, 2
    form = fp8 if eight else lambda w: w.to(torch.bfloat16).to(DEV)
    gate, up, down = form(rand(1, E, ff, D, std=D**-0.5)), form(rand(2, E, ff, D, std=D**-0.5)), form(rand(3, E, D, ff, std=ff**-0.5))
    router = TopKRouter(rand(4, E, D, std=D**-0.5).to(torch.bfloat16).to(DEV), None, top, scoring="sigmoid")
    make = lambda *w: FewTokenExperts(router, *w, "clamped_swish", limit=LIMIT, slope=SLOPE)  # noqa: E731
    x = rand(T, T, D).to(torch.bfloat16).to(DEV)
    want = make(gate, up, down)(x, wide=True)
    assert torch.isfinite(want).all()
    ids = (x.double() @ router.weight.double().t()).topk(top).indices
    hit = (ids == ids[0, 0]).any(1)
    e = int(ids[0, 0])
    for bad in ((spoil(gate, e, 70, 3), up), (gate, spoil(up, e, 5, 135))):
        got = make(*bad, down)(x, wide=True)  # every output of the expert adds every inner number
        assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])
    for value in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[0, 9] = value
        got = make(gate, up, down)(y, wide=True)
        assert torch.equal(got[1:], want[1:])
        if eight or value != value:  # over 16 bits an infinity gives what the formula gives, which may be a number
            assert torch.isnan(got[0]).all()


@pytest.mark.parametrize("T", [1, 40, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_feed_forward_and_experts_of_16_and_32_bits(T, dtype):
    D, ff, E = 128, 96, 4
    w = lambda seed, *shape: rand(seed, *shape, std=shape[-1] ** -0.5).to(dtype).to(DEV)  # noqa: E731
    x = rand(T, T, D).to(dtype).to(DEV)
    gate, up, down = w(1, ff, D), w(2, ff, D), w(3, D, ff)
    dense = lambda g, u: GatedMLP(g, u, down, "clamped_swish", limit=LIMIT, slope=SLOPE)(x)  # noqa: E731
    assert torch.isfinite(dense(gate, up)).all()
    assert torch.isnan(dense(spoil(gate, 3, 5), up)).all() and torch.isnan(dense(gate, spoil(up, 90, 127))).all()
    router = TopKRouter(w(4, E, D), None, E, scoring="sigmoid")
    gates, ups, downs = w(5, E, ff, D), w(6, E, ff, D), w(7, E, D, ff)
    experts = lambda g, u: MixtureOfExperts(router, g, u, downs, "clamped_swish", limit=LIMIT, slope=SLOPE)(x)  # noqa: E731
    assert torch.isfinite(experts(gates, ups)).all()
    assert torch.isnan(experts(spoil(gates, 2, 3, 5), ups)).all() and torch.isnan(experts(gates, spoil(ups, 0, 95, 127))).all()
