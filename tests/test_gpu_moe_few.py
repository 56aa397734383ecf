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
    """-> (y, tolerance before the last rounding, every token's smallest gap of a choice over that gap's own uncertainty)"""
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
    gaps = torch.full((T,), float("inf"), dtype=torch.float64)
    for t in range(T):
        gap = float("inf")
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
        order, gaps[t] = order[:top], gap
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
    return y, tol, gaps


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
    y, tol, gaps = ref
    decided = gaps > 1  # of a token whose choice is closer than fp32 can tell, either choice is right
    assert decided.double().mean() >= 0.9 or not len(decided)
    got = layer(h, wide=wide)
    assert got.shape == y.shape and got.dtype == (torch.float32 if wide else torch.bfloat16)
    tol = tol + torch.finfo(got.dtype).eps / 2 * 1.001 * (y.abs() + tol) + 1e-37
    off = (got.double().cpu() - y).abs()
    off, tol = off[decided], tol[decided]
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


def bf(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(torch.bfloat16).to(DEV)


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,D,ff,E,top", [
    # inner rows in several parts; all tokens on one expert, in several groups; more router outputs than a cluster takes at once; the widest rows
    (1, 64, 6500, 2, 1), (12, 136, 3300, 3, 2), (32, 72, 1700, 1, 1), (32, 72, 100, 2, 2), (3, 64, 40, 300, 2), (20, 264, 40, 140, 7), (2, 11264, 40, 2, 1),
])
def test_long_crowded_and_wide(T, D, ff, E, top, fp8):
    h, router, wg, wu, wd = make(T, D, ff, E, fp8)
    check(FewTokenExperts(TopKRouter(router, None, top), wg, wu, wd, "silu"), h, reference(h, router, wg, wu, wd, "silu", top=top))


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T,scoring,groups,identity,act,gated", [
    (3, "sigmoid", None, 0, "gelu_tanh", True), (12, "softmax_all", None, 2, "silu", True), (6, "softmax_all", (4, 2), 0, "clamped_swish", True),
    (20, "softmax", (3, 1), 1, "silu", False), (8, "sigmoid", None, 0, "relu_squared", False), (27, "softmax", None, 0, "relu_squared", False),
])
def test_routers_and_activations(T, scoring, groups, identity, act, gated, fp8):
    D, ff, E, top = 144, 88, 12 - identity, 3
    h, router, wg, wu, wd = make(T, D, ff, E, fp8, gated=gated, identity=identity, seed=3)
    gen = torch.Generator().manual_seed(T)
    bias = bf(gen, E + identity, std=0.5)
    all_scores = scoring == "softmax_all"
    choice = bf(gen, E + identity, std=0.1) if all_scores else None
    limit, slope = (1.2, 1.7) if act == "clamped_swish" else (0.0, 1.0)
    r = TopKRouter(router, bias, top, scoring=scoring, choice_bias=choice, weight_scale=2.5 if all_scores else 1.0, groups=groups)
    layer = FewTokenExperts(r, wg, wu, wd, act, identity=identity, limit=limit, slope=slope)
    ref = reference(h, router, wg, wu, wd, act, scoring, bias, choice, 2.5 if all_scores else 1.0, groups, top, identity, limit, slope)
    check(layer, h, ref)


@gpu
@pytest.mark.parametrize("T", [0, 1, 32, 33, 70])
def test_shared_expert_and_runs(T):
    D, ff, E, top = 96, 48, 10, 2
    h, router, wg, wu, wd = make(T, D, ff, E, True, seed=5)
    gen = torch.Generator().manual_seed(T + 1)
    shared = GatedMLP(bf(gen, 40, D, std=D**-0.5), bf(gen, 40, D, std=D**-0.5), bf(gen, D, 40, std=40**-0.5), "silu")
    side = bf(gen, 1, D, std=D**-0.5)
    layer = FewTokenExperts(TopKRouter(router, None, top), wg, wu, wd, "silu", shared, shared_gate=side)
    assert layer.run == 32
    y, tol, gap = reference(h, router, wg, wu, wd, "silu", top=top)
    if T:
        s, z = shared(h).double().cpu(), h.double().cpu() @ side.double().cpu().t()
        y = y + torch.sigmoid(z) * s
        tol = tol + (adds(D) * (h.double().cpu().abs() @ side.double().cpu().abs().t()) + 40 * U) * s.abs() + 4 * U * y.abs()
    check(layer, h, (y, tol, gap))


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D,ff", [(5, 3), (100, 50), (203, 77)])
def test_widths_of_no_whole_pieces(D, ff, fp8):
    h, router, wg, wu, wd = make(4, D, ff, 6, fp8, seed=7)
    layer = FewTokenExperts(TopKRouter(router, None, 2), wg, wu, wd, "silu")
    check(layer, h, reference(h, router, wg, wu, wd, "silu", top=2))
    unaligned = torch.cat([h.flatten(), h.new_zeros(8)])[1 : 1 + 3 * D].reshape(3, D)
    assert torch.equal(layer(unaligned.clone()), layer(unaligned))


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [5, 14, 30])
def test_a_token_does_not_depend_on_the_others(T, fp8):
    """Nor on experts that others chose: a token of NaN, and an expert of NaN that one token chooses, spoil these tokens alone."""
    D, ff, E, top = 256, 136, 16, 2
    h, router, wg, wu, wd = make(T, D, ff, E, fp8, seed=11)
    layer = FewTokenExperts(TopKRouter(router, None, top), wg, wu, wd, "silu")
    want = layer(h, wide=True)
    order = torch.randperm(T, generator=torch.Generator().manual_seed(T)).to(DEV)
    x = h[order].contiguous()
    x[0] = float("nan")
    got = layer(x, wide=True)
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], want[order][1:])
    ids = (h.double() @ router.double().t()).topk(top).indices
    e = int(ids[0, 0])
    (wd.values.view(torch.uint8)[e].fill_(0x7F) if fp8 else wd[e].fill_(float("nan")))
    hit = (ids == e).any(1)
    spoiled = layer(h, wide=True)
    assert torch.isnan(spoiled[hit]).all() and torch.equal(spoiled[~hit], want[~hit])


@gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_far_experts_and_large_numbers(fp8):
    """Offsets past 2^31 bytes, and activations and inner rows far from one."""
    D, ff, E = 4096, 2048, 300 if fp8 else 150
    h, router, _, _, _ = make(6, D, 64, 4, False, seed=2)
    gen = torch.Generator(device=DEV).manual_seed(1)
    stacks = []
    for shape in ((E, ff, D), (E, ff, D), (E, D, ff)):
        w = torch.empty(shape, dtype=torch.uint8 if fp8 else torch.bfloat16, device=DEV)
        for e in range(E):
            w[e] = torch.randint(0x28, 0x38, shape[1:], generator=gen, device=DEV, dtype=torch.uint8) if fp8 else torch.randn(shape[1:], generator=gen, device=DEV).to(torch.bfloat16) * shape[2] ** -0.5
        stacks.append(Fp8Weights(w.view(torch.float8_e4m3fn), torch.full((E, shape[1] // 128, shape[2] // 128), 0.02, device=DEV)) if fp8 else w)
    assert E * ff * D * (1 if fp8 else 2) > 2**31
    bias = torch.arange(E, dtype=torch.float32).to(torch.bfloat16).to(DEV)  # the last ones, apart by more than their rounding
    r = torch.zeros(E, D, dtype=torch.bfloat16, device=DEV)
    bias[: E - 3] = -100
    bias[E - 3 :] = torch.tensor([1.0, 2.0, 3.0])
    layer = FewTokenExperts(TopKRouter(r, bias, 2), *stacks, "silu")
    last = [Fp8Weights(s.values[E - 2 :], s.scales[E - 2 :]) if fp8 else s[E - 2 :].clone() for s in stacks]
    for scale in (1.0, 2.0**40, 2.0**-30):
        x = (h.float() * scale).to(torch.bfloat16)
        small = FewTokenExperts(TopKRouter(r[E - 2 :].clone(), bias[E - 2 :].clone(), 2), *last, "silu")
        assert torch.equal(layer(x, wide=True), small(x, wide=True))
        ref = reference(x, r[E - 2 :], *last, "silu", bias=bias[E - 2 :], top=2)
        check(layer, x, ref)


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("T", [1, 20])
def test_captured_and_on_two_streams(T, fp8):
    D, ff, E, top = 512, 264, 24, 4
    h, router, wg, wu, wd = make(T, D, ff, E, fp8, seed=13)
    layer = FewTokenExperts(TopKRouter(router, None, top), wg, wu, wd, "silu")
    inputs = [torch.roll(h, 8 * i, 1).contiguous() for i in range(6)]
    want = [layer(x) for x in inputs]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        x = inputs[i].clone()
        layer(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(x)
        graphs.append((g, x, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(12):
        for (g, x, out), s, k in zip(graphs, streams, (turn % 6, (turn + 3) % 6)):
            with torch.cuda.stream(s):
                x.copy_(inputs[k])
                g.replay()
        torch.cuda.synchronize()
        for (g, x, out), k in zip(graphs, (turn % 6, (turn + 3) % 6)):
            assert torch.equal(out, want[k])
    got = {}
    for turn in range(6):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[turn, j] = layer(inputs[turn])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[turn]) for (turn, _), y in got.items())


@gpu
def test_a_block_of_8_bit_layers_in_one_graph():
    """Projection, feed-forward and experts of 8 bits as a decoding step runs them: each against its own input, eager and replayed."""
    from tests import test_gpu_fp8 as f8
    from tiny_llm_b200.fp8 import fp8_linear
    from tiny_llm_b200.mlp import Fp8GatedMLP

    T, D = 6, 384
    x, w, _ = f8.make(T, D, 200, torch.bfloat16)
    gate, up, down = f8.make(1, 520, D, torch.bfloat16, seed=1)[1], f8.make(1, 520, D, torch.bfloat16, seed=2)[1], f8.make(1, D, 520, torch.bfloat16, seed=3)[1]
    dense = Fp8GatedMLP(gate, up, down, "silu")
    _, router, eg, eu, ed = make(T, D, 136, 10, True, seed=17)
    experts = FewTokenExperts(TopKRouter(router, None, 3), eg, eu, ed, "silu")

    def step(v):
        a = fp8_linear(v, w)
        b = dense(a)
        return a, b, experts(b)

    eager = step(x)
    f8.check_linear(x, w, None, eager[0])
    f8.check_mlp(eager[0], gate, up, down, "silu", eager[1])
    check(lambda h, wide: experts(h, wide=wide), eager[1], reference(eager[1], router, eg, eu, ed, "silu", top=3))
    held = x.clone()
    g = torch.cuda.CUDAGraph()
    step(held)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = step(held)
    for shift in (0, 3, 7):
        held.copy_(torch.roll(x, shift, 1))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(held)))


@gpu
def test_a_model_runs_its_experts_in_two_launches():
    """The same greedy continuation and logits within the rounding of bf16 activations, with the option and without."""
    from tiny_llm_b200 import greedy_generate_ids
    from tiny_llm_b200.models import model_class
    from tiny_llm_b200.synthetic import synthetic_voluzen, voluzen_config

    from tests import test_gpu_voluzen as V

    config = voluzen_config(pattern="CSM", experts=8, top=2, expert_ff=64)
    tensors = V.decisive_routers(synthetic_voluzen(config, seed=5))
    prompt = [3, 17, 5, 99, 42, 7]
    models = [model_class("Voluzen")(config, tensors, few_token_experts=few) for few in (False, True)]
    assert all(layer.mlp.few is not None for layer in models[1].layers if layer.mlp is not None and hasattr(layer.mlp, "few"))
    logits = []
    for model in models:
        cache = model.create_kv_cache()
        logits.append(model(torch.tensor([prompt], device=DEV), 0, cache)[0].double().cpu())
    assert V.rows_match(logits[1], logits[0], torch.bfloat16)
    before = __import__("extensions_b200.tiny_llm_ext_b200.blocks", fromlist=["x"]).launch_count()
    assert len(greedy_generate_ids(models[1], prompt, 5)) >= 5
    assert __import__("extensions_b200.tiny_llm_ext_b200.blocks", fromlist=["x"]).launch_count() > before
