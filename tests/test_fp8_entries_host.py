"""The extension's own entries of the 8-bit products look at the matrix they are given, ahead of anything that reads it."""

import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks

F8 = torch.float8_e4m3fn


def values(n, k):
    return torch.zeros(n, k, dtype=F8)


@pytest.mark.parametrize("w,scales", [
    (torch.zeros(8, 16, dtype=torch.uint8), torch.ones(1, 1)),
    (values(8, 15), torch.ones(1, 1)),
    (values(16, 8).t(), torch.ones(1, 1)),
    (values(16, 16)[None], torch.ones(1, 1)),
    (values(8, 16), torch.ones(1)),
    (values(8, 16), torch.ones(1, 1, dtype=torch.float64)),
    (values(129, 16), torch.ones(1, 1)),
    (values(129, 16), torch.ones(4, 1)[::2]),
])
def test_a_matrix_of_another_form_is_refused(w, scales):
    with pytest.raises(RuntimeError, match="values must be|scales must be"):
        blocks.fp8_linear(torch.zeros(2, 16), w, scales, 16)


def test_feed_forwards_of_other_forms_are_refused():
    x, good = torch.zeros(2, 16), ((values(512, 16), torch.ones(4, 1)), (values(16, 144), torch.ones(1, 2)))
    with pytest.raises(RuntimeError, match="GPU-only"):  # the forms are right: the device is not
        blocks.fp8_gated_mlp(x, *good, 16, 130, blocks.ACT_SILU)
    for gate_up, down in (((values(256, 16), torch.ones(2, 1)), good[1]), (good[0], (values(16, 112), torch.ones(1, 1))), (good[0], (values(15, 144), torch.ones(1, 2))),
                          ((good[0][0], torch.ones(4, 2)), good[1]), (good[0], (good[1][0], torch.ones(2, 1)))):
        with pytest.raises(RuntimeError, match="values must be|scales must be"):
            blocks.fp8_gated_mlp(x, gate_up, down, 16, 130, blocks.ACT_SILU)


@pytest.mark.gpu
def test_scales_on_another_device_are_refused():
    with pytest.raises(RuntimeError, match="scales must be"):
        blocks.fp8_linear(torch.zeros(2, 16, device="cuda"), values(8, 16).cuda(), torch.ones(1, 1), 16)
