"""8-bit weights and the few-token experts where no GPU is needed: the form and its checks, what the layers and the C entry points refuse."""

import ctypes

import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks
from tiny_llm_b200 import Fp8Weights, fp8_linear
from tiny_llm_b200.fp8 import BLOCK, interleaved
from tiny_llm_b200.mlp import FewTokenExperts, Fp8GatedMLP, MixtureOfExperts, TopKRouter


def weights(*shape, seed=0):
    return Fp8Weights.from_tensor(torch.randn(*shape, generator=torch.Generator().manual_seed(seed)))


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 17), (3, 200, 300), (2, 2, 5, 129)])
def test_rounding_and_what_it_stands_for(shape):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(1)) * 3
    q = Fp8Weights.from_tensor(w)
    n, k = shape[-2:]
    assert q.shape == shape and q.scales.shape == (*shape[:-2], -(-n // BLOCK), -(-k // BLOCK)) and q.values.shape[-1] % 16 == 0
    assert (q.values[..., k:].float() == 0).all()
    got = q.dequantize()
    wide = q.scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    # half a step of three bits, or half of the smallest step, and the roundings of the scale, the quotient and the product
    assert ((got - w).abs() <= 2.0**-4 * w.abs() * (1 + 2.0**-20) + 2.0**-10 * wide * (1 + 2.0**-20)).all()
    assert (q.dequantize(torch.float64).float() - got).abs().max() == 0


def test_numbers_of_a_checkpoint_stay_as_they_are():
    raw = torch.randint(0, 0x7E, (200, 48), dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.rand(2, 1)
    w = Fp8Weights(raw, scales)
    assert w.values.data_ptr() == raw.data_ptr()  # whole 16-byte rows: no copy
    w = Fp8Weights(raw[:, :45], scales)
    assert torch.equal(w.values[:, :45].view(torch.uint8), raw[:, :45].view(torch.uint8)) and (w.values[:, 45:].view(torch.uint8) == 0).all()


@pytest.mark.parametrize("make", [
    lambda: Fp8Weights(torch.zeros(4, 4), torch.ones(1, 1)),
    lambda: Fp8Weights(torch.zeros(4, dtype=torch.float8_e4m3fn), torch.ones(1)),
    lambda: Fp8Weights(torch.zeros(0, 4, dtype=torch.float8_e4m3fn), torch.ones(0, 1)),
    lambda: Fp8Weights(torch.zeros(129, 4, dtype=torch.float8_e4m3fn), torch.ones(1, 1)),
    lambda: Fp8Weights(torch.zeros(4, 4, dtype=torch.float8_e4m3fn), torch.ones(1, 1, dtype=torch.float64)),
    lambda: Fp8Weights.from_tensor(torch.tensor([[1.0, float("inf")]])),
    lambda: Fp8Weights.from_tensor(torch.tensor([[1.0, float("nan")]])),
    lambda: Fp8Weights.from_tensor(torch.tensor([[1, 2]])),
    lambda: Fp8GatedMLP(weights(8, 16), weights(9, 16), weights(16, 8), "silu"),
    lambda: Fp8GatedMLP(weights(8, 16), weights(8, 16), weights(8, 16), "silu"),
    lambda: Fp8GatedMLP(weights(8, 16), weights(8, 16), weights(16, 8), "relu_squared"),
    lambda: Fp8GatedMLP(weights(8, 16), weights(8, 16), weights(16, 8), "clamped_swish"),
    lambda: Fp8GatedMLP(torch.zeros(8, 16), weights(8, 16), weights(16, 8), "silu"),
    lambda: fp8_linear(torch.zeros(2, 16), weights(3, 8, 16)),
])
def test_refused_with_a_value_error(make):
    with pytest.raises(ValueError):
        make()


def test_cpu_tensors_are_refused():
    for call in (lambda: fp8_linear(torch.zeros(2, 16), weights(8, 16)), lambda: fp8_linear(torch.zeros(2, 15), weights(8, 16)),
                 lambda: Fp8GatedMLP(weights(8, 16), weights(8, 16), weights(16, 8), "silu")(torch.zeros(2, 16))):
        with pytest.raises(RuntimeError):
            call()


def stack(fp8=False, E=4, ff=8, D=16, router_outputs=None, dtype=torch.bfloat16):
    w = [torch.randn(*s, generator=torch.Generator().manual_seed(2)) for s in ((E, ff, D), (E, ff, D), (E, D, ff))]
    w = [Fp8Weights.from_tensor(x) for x in w] if fp8 else [x.to(dtype) for x in w]
    return TopKRouter(torch.zeros(router_outputs or E, D, dtype=dtype), None, 2), *w


@pytest.mark.parametrize("make", [
    lambda: FewTokenExperts(*stack(router_outputs=5), "silu"),
    lambda: FewTokenExperts(*stack(dtype=torch.float32), "silu"),
    lambda: FewTokenExperts(*stack(), "relu_squared"),
    lambda: FewTokenExperts(*stack(), "clamped_swish"),
    lambda: FewTokenExperts(*stack()[:3], stack()[1], "silu"),
    lambda: FewTokenExperts(*stack()[:3], stack(fp8=True)[3], "silu"),
    lambda: FewTokenExperts(*stack(), "silu", shared_gate=torch.zeros(1, 16, dtype=torch.bfloat16)),
    lambda: MixtureOfExperts(stack()[0], None, *stack()[2:], "relu_squared", weight_on="input").use_few_tokens(),
])
def test_layers_of_experts_are_checked(make):
    with pytest.raises(ValueError):
        make()


@pytest.mark.parametrize("fp8", [False, True])
def test_experts_on_the_cpu_are_refused(fp8):
    with pytest.raises(RuntimeError):
        FewTokenExperts(*stack(fp8=fp8), "silu")


def test_interleaved_halves():
    gate, up = weights(130, 20, seed=3), weights(130, 20, seed=4)
    values, scales = interleaved(gate, up)
    raw = values.view(torch.uint8).reshape(2, 2, 128, 32)
    for half, w in enumerate((gate, up)):
        joined = raw[:, half].reshape(256, 32)
        assert torch.equal(joined[:130], w.values.view(torch.uint8)) and (joined[130:] == 0).all()
        assert torch.equal(scales.reshape(2, 2, 1)[:, half], w.scales)


def test_how_many_tokens_a_call_takes():
    few = blocks.moe_few_tokens
    assert few(2048, 64, 64, 6, 0, True) == 32 and few(2048, 64, 64, 6, 0, False) == 32
    assert 0 < few(8192, 64, 64, 6) < 32 and few(1 << 20, 64, 64, 6) == 0
    assert few(2048, 1025, 1025, 6) == 0 and few(2048, 64, 65, 6) == 0 and few(2048, 64, 64, 65) == 0 and few(0, 64, 64, 6) == 0
    assert few(256, 512, 512, 64) == 8  # at most 512 pairs


def test_c_entries_report_bad_arguments_without_a_device():
    lib = blocks.library()
    one = ctypes.c_void_p(4096)  # never read
    linear = lambda **k: lib.tlb_fp8_linear(*({"x": one, "ldx": 64, "w": one, "ldw": 64, "sw": one, "bias": None, "out": one, "rows": 2, "n": 8, "k": 64, "ws": one,  # noqa: E731
                                               "bytes": 1 << 20, "dtype": 2, "stream": None} | k).values())
    for bad in (dict(x=None), dict(w=None), dict(sw=None), dict(out=None), dict(ws=None), dict(n=0), dict(k=0), dict(ldx=63), dict(ldw=48), dict(ldw=72), dict(dtype=1),
                dict(bytes=3), dict(w=ctypes.c_void_p(4104)), dict(ws=ctypes.c_void_p(4097))):
        assert linear(**bad) < 0 and lib.tlb_last_error()
    assert linear(rows=0) == 0
    mlp = lambda **k: lib.tlb_fp8_gated_mlp(*({"x": one, "ldx": 64, "wg": one, "ldg": 64, "sg": one, "wd": one, "ldd": 32, "sd": one, "out": one, "rows": 2, "dim": 64,  # noqa: E731
                                               "ff": 32, "act": 0, "limit": 0.0, "slope": 1.0, "ws": one, "bytes": 1 << 20, "dtype": 2, "stream": None} | k).values())
    for bad in (dict(x=None), dict(wg=None), dict(wd=None), dict(act=2), dict(act=3), dict(ff=0), dict(ldd=16), dict(ldg=60), dict(bytes=8), dict(dtype=1)):
        assert mlp(**bad) < 0 and lib.tlb_last_error()
    base = dict(router=4096, w_gate=4096, w_up=4096, w_down=4096, s_gate=4096, s_up=4096, s_down=4096, dim=64, outputs=8, experts=8, top=2, fp8=1, ff=32, ld_in=64, ld_out=32,
                weight_scale=1.0)

    def few(tokens=2, x=one, shared=None, out=one, ws=one, size=1 << 20, **k):
        layer = blocks.FewLayer(**(base | k))
        return lib.tlb_moe_few(ctypes.addressof(layer), x, tokens, shared, out, 0, ws, size, None)

    for bad in (dict(x=None), dict(out=None), dict(ws=None), dict(size=64), dict(tokens=33), dict(router=None), dict(w_up=None), dict(s_up=None), dict(dim=60), dict(ld_in=48),
                dict(ld_out=24), dict(act=2), dict(act=3), dict(scoring=3), dict(group_count=3, group_keep=1), dict(group_count=8, group_keep=1), dict(top=9), dict(experts=9),
                dict(side_w=4096), dict(w_down=4100), dict(ff=0)):
        assert few(**bad) < 0 and lib.tlb_last_error()
    assert few(tokens=0) == 0
