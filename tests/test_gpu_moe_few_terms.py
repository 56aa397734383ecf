"""What the experts for few tokens keep of a number.

A number meets weights of 8 or 16 bits as several terms, a column of a product each: each of these tests looks at one number by itself, so that a term that is left out, has
another weight or stands in another column is an error of its whole size.  One choice of each token has the weight 1 (the softmax of one logit), and a matrix with
one entry 1 a row hands single numbers on.

u = 2^-24.  An inner number silu(v) v' is off by some rounded operations: 40 u of itself covers the exponential (2 ulp), the sum, the quotient and the products."""

import pytest
import torch

from tiny_llm_b200.fp8 import Fp8Weights
from tiny_llm_b200.mlp import FewTokenExperts, TopKRouter

from tests.test_gpu_moe_few import make

DEV = "cuda"
U = 2.0**-24
pytestmark = pytest.mark.gpu


def picks(rows, cols, seed, eight, experts=2):
    """``[experts, rows, cols]`` with one entry 1 a row -> (the matrix, the columns)."""
    at = torch.randint(0, cols, (experts, rows), generator=torch.Generator().manual_seed(seed))
    w = torch.nn.functional.one_hot(at, cols).to(torch.bfloat16).to(DEV)
    if eight:
        w = Fp8Weights(w.to(torch.float8_e4m3fn), torch.ones(experts, -(-rows // 128), -(-cols // 128), device=DEV))
    return w, at


def routed(T, D, seed):
    """A router of two experts that takes either for some tokens, by channel 0, which all tokens have large."""
    weight = torch.zeros(2, D, dtype=torch.bfloat16, device=DEV)
    weight[0, 0] = 1
    return TopKRouter(weight, None, 1), (torch.arange(T) % 2 == 0)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T,D,ff", [(1, 64, 40), (2, 72, 200), (8, 256, 130), (17, 136, 300), (32, 200, 520)])
def test_an_output_that_is_one_inner_number(T, D, ff, eight):
    gen = torch.Generator().manual_seed(T)
    x = torch.randn(T, D, generator=gen)
    router, first = routed(T, D, 1)
    x[:, 0] = torch.where(first, 1.0, -1.0)
    x = x.to(torch.bfloat16)
    up, of_x = picks(ff, D, 2, eight)
    down, of_inner = picks(D, ff, 3, eight)
    layer = FewTokenExperts(router, None, up, down, "silu")
    got = layer(x.to(DEV), wide=True).double().cpu()
    rounded = layer(x.to(DEV)).double().cpu()
    e = torch.where(first, 0, 1)
    v = x.double()
    v = torch.gather(v, 1, of_x[e])  # [T, ff]
    inner = torch.nn.functional.silu(v)
    want = torch.gather(inner, 1, of_inner[e])
    # fp32 numbers: three bf16 terms hold all 24 bits.  Six e4m3 terms leave 2^-24 of a number (2^-4 each), or half of the smallest step of the sixth, which is
    # 2^-10 / 16^5 where the largest of the block is scaled to 2^7 at least: 2^-37 of it.  The terms are added one after another: a rounding each.
    tol = (40 + 8) * U * inner.abs()
    if eight:
        # A token's largest is scaled to 2^7 at least, and the second of its two e4m3 terms ends at 2^-9 / 16.  The 8 bits of an entry reach 2^-7 of it down: from 2^-6 on, which is
        # 2^-13 of the largest, it is held as it is, below it to half of that step, 2^-14 or 2^-21 of the largest.  |silu'| <= 1.1
        largest = x.double().abs().amax(1, keepdim=True)
        tol = tol + 2.0**-37 * inner.abs().amax(1, keepdim=True) + torch.where(v.abs() < 2.0**-13 * largest, 1.1 * 2.0**-21 * largest, 0.0)
    tol = torch.gather(tol, 1, of_inner[e])
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()
    # bf16 outputs over 8-bit experts: three e4m3 terms leave 2^-12 of an inner number and 2^-10 / 16^2 / 2^7 = 2^-25 of its block's largest
    less = tol + want.abs() * (2.0**-12 if eight else 0) + (2.0**-25 * inner.abs().amax(1, keepdim=True) if eight else 0)
    assert ((rounded - want).abs() <= less + 2.0**-8 * (want.abs() + less)).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T", [1, 5, 20, 32])
def test_numbers_of_a_token_far_below_its_largest(T, eight):
    """Channels that span 2^40.  Over 16-bit experts they are what they are; over 8-bit ones what lies below 2^-21 of the token's largest magnitude is lost."""
    D = ff = 256
    gen = torch.Generator().manual_seed(T)
    x = torch.randn(T, D, generator=gen) * torch.exp2(-40 * torch.rand(T, D, generator=gen))
    router, first = routed(T, D, 1)
    x[:, 0] = torch.where(first, 4.0, -4.0)
    x = x.to(torch.bfloat16)
    up, of_x = picks(ff, D, 5, eight)
    down, of_inner = picks(D, ff, 6, eight)
    got = FewTokenExperts(router, None, up, down, "silu")(x.to(DEV), wide=True).double().cpu()
    e = torch.where(first, 0, 1)
    v = torch.gather(x.double(), 1, of_x[e])
    inner = torch.nn.functional.silu(v)
    want = torch.gather(inner, 1, of_inner[e])
    tol = 48 * U * want.abs()
    if eight:  # |silu'| <= 1.1; and the inner numbers' own terms, against the largest of the block
        lost = 1.1 * 2.0**-21 * x.double().abs().amax(1, keepdim=True)
        tol = tol + lost + 2.0**-37 * (inner.abs().amax(1, keepdim=True) + lost)
    assert ((got - want).abs() <= tol + 1e-37).all()
