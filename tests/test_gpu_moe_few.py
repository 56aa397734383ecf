"""A mixture-of-experts layer for a few tokens in two launches against float64: token counts around the kernels' tiles, widths that end inside a
block, one expert to many, every scoring, identity and shared experts, weights of 16 and of 8 bits.

The tolerance follows the arithmetic.  With u = 2^-24: a sum of n products through the tensor cores' products of 16 and the warps' shares is off by at most
(n / 16 + 40) 2u of the sum of magnitudes; x as fp16 by 2^-24 of its row's largest; an inner number by 2^-11 of itself or 2^-24 of its row's largest; |silu'| <= 1.1."""

import pytest
import torch

from tiny_llm_b200.fp8 import BLOCK, Fp8Weights
from tiny_llm_b200.mlp import FewTokenExperts, GatedMLP, TopKRouter

DEV = "cuda"
gpu = pytest.mark.gpu
U = 2.0**-24


def weights64(w, k):
    if not isinstance(w, Fp8Weights):
        return w.double().cpu()
    n = w.shape[-2]
    wide = w.scales.double().cpu().repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return w.values[..., :k].float().double().cpu() * wide


def adds(n):
    return (n / 16 + 40) * 2 * U


def reference(h, router, wg, wu, wd, act, scoring="softmax", bias=None, choice_bias=None, scale=1.0, groups=None, top=2, identity=0, limit=0.0, slope=1.0):
    """-> (y, tolerance before the last rounding, smallest gap of a choice over its own uncertainty)"""
    x = h.double().cpu()
    T, D = x.shape
    E, ff, _ = wu.shape
    wu64, wd64 = weights64(wu, D), weights64(wd, ff)
    wg64 = None if wg is None else weights64(wg, D)
    r64 = router.double().cpu()
    z = x @ r64.t()
    dz = adds(D) * (x.abs() @ r64.abs().t()) + 4 * U * z.abs()
    if bias is not None:
        z = z + bias.double().cpu()
        dz = dz + 2 * U * z.abs()
    y, tol = torch.zeros(T, D, dtype=torch.float64), torch.zeros(T, D, dtype=torch.float64)
    gap = float("inf")
    for t in range(T):
        score, ds = z[t], dz[t]
        if scoring == "softmax_all":
            p = torch.softmax(z[t], 0)
            dp = p * (2 * dz[t].max() + 40 * U)
            score, ds = p + (0 if choice_bias is None else choice_bias.double().cpu()), dp + 2 * U
        pick = score.clone()
        if groups is not None:
            count, keep = groups
            best = score.reshape(count, -1).max(1).values
            order = best.argsort(descending=True)
            gap = min(gap, ((best[order[keep - 1]] - best[order[keep]]) / (2 * ds.max())).item()) if keep < count else gap
            for j in order[keep:].tolist():
                pick.reshape(count, -1)[j] = -torch.inf
        order = sorted(range(len(pick)), key=lambda e: (-pick[e].item(), e))
        if top < len(pick):
            gap = min(gap, ((pick[order[top - 1]] - pick[order[top]]) / (2 * ds.max())).item())
        order = order[:top]
        if scoring == "softmax":
            w, dw = torch.softmax(z[t, order], 0), 2 * dz[t].max() + 40 * U
        elif scoring == "sigmoid":
            w, dw = torch.sigmoid(z[t, order]), dz[t].max() + 40 * U
        else:
            w = torch.softmax(z[t], 0)[order]
            w, dw = w / w.sum() * scale, 4 * dz[t].max() + 100 * U
        dx = 2 * U * x[t].abs().max()
        for k, e in enumerate(order):
            if e >= E:
                y[t] += w[k] * x[t]
                tol[t] += (dw + 4 * U) * (w[k] * x[t]).abs()
                continue
            up = wu64[e] @ x[t]
            dup = adds(D) * (wu64[e].abs() @ x[t].abs()) + dx * wu64[e].abs().sum(1)
            if wg64 is not None:
                g = wg64[e] @ x[t]
                dg = adds(D) * (wg64[e].abs() @ x[t].abs()) + dx * wg64[e].abs().sum(1)
                if act == "clamped_swish":
                    gc, uc = g.clamp(max=limit), up.clamp(-limit, limit) + 1
                    inner = gc * torch.sigmoid(slope * gc) * uc
                    dinner = 1.1 * max(1.0, slope) * dg * uc.abs() + (gc * torch.sigmoid(slope * gc)).abs() * dup + 40 * U * inner.abs()
                else:
                    f = torch.nn.functional.silu if act == "silu" else lambda v: torch.nn.functional.gelu(v, approximate="tanh")
                    inner = f(g) * up
                    # the hyperbolic tangent of a large negative number cancels against 1: its error is an absolute one
                    dinner = 1.2 * dg * up.abs() + f(g).abs() * dup + 40 * U * inner.abs() + (8 * U * g.abs() * up.abs() if act == "gelu_tanh" else 0)
            elif act == "relu_squared":
                inner = torch.relu(up).square()
                dinner = 2 * torch.relu(up) * dup + dup.square() + 8 * U * inner
            else:
                inner = torch.nn.functional.silu(up)
                dinner = 1.1 * dup + 40 * U * inner.abs()
            dinner = dinner + 2.0**-11 * inner.abs() + 2 * U * inner.abs().max()
            y[t] += w[k] * (wd64[e] @ inner)
            most = wd64[e].abs() @ inner.abs()
            tol[t] += w[k] * (wd64[e].abs() @ dinner + (adds(ff) + dw + 8 * U) * most) + 8 * U * (w[k] * most)
    return y, tol, gap


def make(T, D, ff, E, fp8, gated=True, identity=0, seed=0):
    gen = torch.Generator().manual_seed(seed * 1000 + T * 31 + D + ff * 7 + E)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    h = (rand(T, D) * torch.exp(rand(D))).to(torch.bfloat16)
    router = (2 * rand(E + identity, D) * D**-0.5).to(torch.bfloat16)
    out = []
    for shape in ((E, ff, D), (E, ff, D), (E, D, ff)):
        w = rand(*shape) * shape[-1] ** -0.5
        if fp8:
            w = Fp8Weights.from_tensor(w)
            out.append(Fp8Weights(w.values[..., : shape[-1]].to(DEV), w.scales.to(DEV)))
        else:
            out.append(w.to(torch.bfloat16).to(DEV))
    return h.to(DEV), router.to(DEV), out[0] if gated else None, out[1], out[2]


def check(layer, h, ref, wide=True):
    y, tol, gap = ref
    assert gap > 1, "the inputs decide no choice"
    got = layer(h, wide=wide)
    assert got.shape == y.shape and got.dtype == (torch.float32 if wide else torch.bfloat16)
    tol = tol + torch.finfo(got.dtype).eps / 2 * 1.001 * (y.abs() + tol) + 1e-37
    off = (got.double().cpu() - y).abs()
    assert bool((off <= tol).all()), f"worst {(off / tol).max().item():.2f} times the tolerance"


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,D,ff,E,top", [
    (1, 8, 8, 1, 1), (1, 64, 40, 4, 2), (2, 200, 136, 8, 3), (3, 128, 128, 5, 5), (7, 264, 72, 6, 2), (8, 136, 264, 16, 4), (9, 96, 200, 4, 1), (16, 256, 144, 20, 8),
    (17, 72, 80, 9, 2), (31, 520, 96, 33, 3), (32, 384, 520, 12, 6), (5, 1096, 712, 20, 3), (1, 2048, 1408, 8, 6),
])
def test_layer(T, D, ff, E, top, fp8):
    h, router, wg, wu, wd = make(T, D, ff, E, fp8)
    layer = FewTokenExperts(TopKRouter(router, None, top), wg, wu, wd, "silu")
    ref = reference(h, router, wg, wu, wd, "silu", top=top)
    check(layer, h, ref)
    check(layer, h, ref, wide=False)
