"""A token whose choices name an expert twice."""

import pytest
import torch

from tiny_llm_b200.mlp import FewTokenExperts, MixtureOfExperts, TopKRouter

from tests.test_gpu_moe_few import make

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 32])
def test_choices_that_name_an_expert_twice(T):
    """With fewer outputs than choices that are not minus infinity, the first of the others comes again: the layer adds it as often as the chain of launches does."""
    D, ff, E, top = 64, 48, 6, 4
    h, router, wg, wu, wd = make(T, D, ff, E, False, seed=6)
    choice = torch.full((E,), float("-inf"), dtype=torch.bfloat16, device=DEV)
    choice[1] = choice[4] = 0
    r = TopKRouter(router, None, top, scoring="softmax_all", choice_bias=choice, weight_scale=2.0)
    ids, weights = r(h)
    assert any(len(set(row)) < top for row in ids.tolist())
    chain = MixtureOfExperts(r, wg, wu, wd, "silu")
    few = FewTokenExperts(r, wg, wu, wd, "silu")(h, wide=True)
    want = torch.zeros(T, D, dtype=torch.float64)
    x = h.double().cpu()
    for t in range(T):
        for e, g in zip(ids[t].tolist(), weights[t].double().tolist()):
            inner = torch.nn.functional.silu(wg[e].double().cpu() @ x[t]) * (wu[e].double().cpu() @ x[t])
            want[t] += g * (wd[e].double().cpu() @ inner)
    # The chain keeps inner rows in bf16 (2^-8 of each, which do not all err alike), the few-token layer's sums are fp32: some 50 operations and the tensor cores' sums of
    # 64 and 48 products, each off by 2^-23 of magnitudes that add up to ten times the outputs at most.  An expert added once in place of three times is off by its own size.
    largest = want.abs().max()
    assert ((chain(h).double().cpu() - want).abs() <= 2.0**-7 * largest).all()  # its inner rows are bf16
    assert ((few.double().cpu() - want).abs() <= 2.0**-14 * largest).all()
