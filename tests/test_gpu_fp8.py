"""Products over 8-bit weights against float64: sizes at the edges of blocks, tiles and reductions, strides, empty inputs, numbers that are none,
streams and captured graphs; the gated feed-forward; the refusals of both.

Tolerance of a product: the products of two e4m3 numbers are exact, a block's 128 of them are added in the tensor cores (an addition is off by at most
2^-23 of what is added, if it cuts), the blocks in fp32 with two roundings each, and the result is rounded to its type once."""

import pytest
import torch

from tiny_llm_b200.fp8 import BLOCK, Fp8Weights, fp8_linear
from tiny_llm_b200.mlp import Fp8GatedMLP

DEV = "cuda"
gpu = pytest.mark.gpu


def nearest_e4m3(v):
    _, e = torch.frexp(v)
    step = torch.exp2(torch.clamp(e.double() - 4, min=-9.0))
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def rounded_rows(x):
    """float64: what the rows stand for once they are e4m3 numbers (scales and products rounded to fp32 as the operator says)."""
    x = x.detach().cpu().float().double()
    out = torch.empty_like(x)
    for k in range(0, x.shape[1], BLOCK):
        part = x[:, k : k + BLOCK]
        most = part.abs().amax(dim=1, keepdim=True)
        most = torch.where(most < 2.0**-100, torch.full_like(most, 2.0**-100), most)
        top = torch.full_like(most, 448.0)
        q = nearest_e4m3((part * (top / most).float().double()).float().double()) * (most / top).float().double()
        out[:, k : k + BLOCK] = torch.where(torch.isfinite(most), q, torch.full_like(q, torch.nan))
    return out


def make(rows, n, k, dtype, seed=0, bias=False):
    gen = torch.Generator().manual_seed(seed + rows * 7 + n * 3 + k)
    x = (torch.randn(rows, k, generator=gen) * torch.exp(torch.randn(k, generator=gen))).to(dtype)
    w = Fp8Weights.from_tensor(torch.randn(n, k, generator=gen) * torch.exp(torch.randn(n, 1, generator=gen)) * k**-0.5)
    return x.to(DEV), Fp8Weights(w.values[:, :k].to(DEV), w.scales.to(DEV)), torch.randn(n, generator=gen).to(dtype).to(DEV) if bias else None


def product_tolerance(rows64, w64, want, dtype):
    """Per entry: see the head of the file; ``rows64`` and ``w64`` are what is multiplied."""
    most = rows64.abs() @ w64.abs().t()
    blocks = -(-rows64.shape[1] // BLOCK)
    return (2 * BLOCK + 3 * blocks + 4) * 2.0**-24 * most + torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + 1e-38


def check_linear(x, w, bias, got):
    xq, w64 = rounded_rows(x), w.dequantize(torch.float64).cpu()
    # dequantize() rounds value * scale to fp32: multiply in 64 bits instead
    n, k = w.shape
    w64 = w.values[:, :k].float().double().cpu() * w.scales.double().cpu().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    want = xq @ w64.t()
    if bias is not None:
        want = want + bias.double().cpu()
    tol = product_tolerance(xq, w64, want, x.dtype)
    if bias is not None:
        tol = tol + 2.0**-23 * (want.abs() + bias.double().cpu().abs())
    assert got.dtype == x.dtype and got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"worst {(off / tol).max().item():.2f} times the tolerance"


@gpu
@pytest.mark.parametrize("rows", [1, 2, 8, 9, 16, 17, 33, 64, 65, 128, 129, 257, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 127), (200, 300), (640, 1000), (333, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(rows, n, k, dtype):
    x, w, bias = make(rows, n, k, dtype, bias=n % 2 == 1)
    check_linear(x, w, bias, fp8_linear(x, w, bias))


@gpu
@pytest.mark.parametrize("rows,k,apart", [(33000, 112, 0), (16400, 144, 16), (11001, 384, 0), (4100, 1040, 8), (4100, 1048, 0), (3700, 1200, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_of_many_rows(rows, k, apart, dtype):
    """Enough rows for the rounding of several runs a warp: runs that end early, rows apart, rows that are no whole pieces."""
    x, w, _ = make(rows, 24, k, dtype)
    if apart:
        wide = torch.zeros(rows, k + apart, dtype=dtype, device=DEV)
        wide[:, :k] = x
        x = wide[:, :k]
    x[7, :] = 0
    x[8, k // 2] = float("inf")
    got = fp8_linear(x, w)
    assert torch.isnan(got[8]).all() and (got[7] == 0).all()
    keep = torch.arange(rows, device=DEV) != 8
    check_linear(x[keep], w, None, got[keep])


@gpu
@pytest.mark.parametrize("n", [4108, 4112, 6001, 6112, 7105, 7120, 8331, 8336])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_of_every_width_of_tile(n, dtype):
    """Tiles of 160, 192, 224 and 256 outputs, whole pieces of a row and not; the tile's width changes no bits."""
    x, w, bias = make(257, n, 300, dtype, bias=n % 2 == 1)
    got = fp8_linear(x, w, bias)
    check_linear(x, w, bias, got)
    part = fp8_linear(x, Fp8Weights(w.values[:4096, :300], w.scales[:32].contiguous()), None if bias is None else bias[:4096].contiguous())
    assert torch.equal(part, got[:, :4096])


@gpu
@pytest.mark.parametrize("rows,n,k", [(1, 2560, 9728), (24, 2560, 4096), (48, 5000, 3000), (100, 2048, 6144), (700, 1200, 2600), (2100, 900, 1111)])
def test_linear_of_real_sizes(rows, n, k):
    x, w, bias = make(rows, n, k, torch.bfloat16)
    check_linear(x, w, bias, fp8_linear(x, w, bias))


def check_mlp(x, gate, up, down, act, got, limit=0.0, slope=1.0):
    """The inner rows are rounded by the operator from its own fp32 sums: an entry next to a border may be rounded the other way, which is one step of its
    run's scale.  So the second product's tolerance counts one step for each inner number that lies within the first product's tolerance of a border."""
    plain = lambda w: w.values[:, : w.shape[1]].float().double().cpu() * w.scales.double().cpu().repeat_interleave(BLOCK, 0)[: w.shape[0]].repeat_interleave(BLOCK, 1)[:, : w.shape[1]]  # noqa: E731
    xq, wg, wu, wd = rounded_rows(x), plain(gate), plain(up), plain(down)
    g, u = xq @ wg.t(), xq @ wu.t()
    blocks = -(-xq.shape[1] // BLOCK)
    sums = (2 * BLOCK + 3 * blocks + 4) * 2.0**-24
    dg, du = sums * (xq.abs() @ wg.abs().t()), sums * (xq.abs() @ wu.abs().t())
    if act == "clamped_swish":
        gc, uc = g.clamp(max=limit), u.clamp(-limit, limit) + 1
        inner, di = gc * torch.sigmoid(slope * gc) * uc, 1.1 * max(1.0, slope) * dg * uc.abs() + (gc * torch.sigmoid(slope * gc)).abs() * du
    else:
        f = torch.nn.functional.silu if act == "silu" else lambda v: torch.nn.functional.gelu(v, approximate="tanh")
        inner, di = f(g) * u, 1.2 * dg * u.abs() + f(g).abs() * du + (8 * 2.0**-24 * g.abs() * u.abs() if act == "gelu_tanh" else 0)
    di = di + 40 * 2.0**-24 * inner.abs()
    low, high, near = torch.empty_like(inner), torch.empty_like(inner), torch.empty_like(inner)
    for k in range(0, inner.shape[1], BLOCK):
        part, d = inner[:, k : k + BLOCK], di[:, k : k + BLOCK]
        most = part.abs().amax(dim=1, keepdim=True).clamp_min(2.0**-100)
        off = (d.amax(dim=1, keepdim=True) / most).clamp_max(1.0) + 4 * 2.0**-24  # the scale's own
        v, dv = part * (448.0 / most), d * (448.0 / most) + 2 * off * part.abs() * (448.0 / most)
        s = most / 448.0
        near[:, k : k + BLOCK] = nearest_e4m3(v) * s
        low[:, k : k + BLOCK], high[:, k : k + BLOCK] = nearest_e4m3(v - dv) * s, nearest_e4m3(v + dv) * s
        spread = off * nearest_e4m3(v).abs() * s
        low[:, k : k + BLOCK] -= spread
        high[:, k : k + BLOCK] += spread
    want = near @ wd.t()
    tol = torch.maximum(high - near, near - low) @ wd.abs().t() + product_tolerance(near, wd, want, x.dtype)
    tol = tol + torch.finfo(x.dtype).eps / 2 * tol
    off = (got.double().cpu() - want).abs()
    assert got.dtype == x.dtype and got.shape == want.shape
    assert bool((off <= tol).all()), f"worst {(off / tol).max().item():.2f} times the tolerance"


@gpu
@pytest.mark.parametrize("rows", [1, 5, 16, 17, 70, 128, 129, 300])
@pytest.mark.parametrize("dim,ff,act", [(16, 1, "silu"), (128, 128, "silu"), (200, 129, "clamped_swish"), (333, 700, "gelu_tanh"), (640, 1400, "silu")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gated_mlp(rows, dim, ff, act, dtype):
    x, gate, _ = make(rows, ff, dim, dtype, seed=1)
    up, down = make(1, ff, dim, dtype, seed=2)[1], make(1, dim, ff, dtype, seed=3)[1]
    layer = Fp8GatedMLP(gate, up, down, act, limit=1.5 if act == "clamped_swish" else 0.0, slope=1.7 if act == "clamped_swish" else 1.0)
    check_mlp(x, gate, up, down, act, layer(x), 1.5, 1.7 if act == "clamped_swish" else 1.0)


@gpu
@pytest.mark.parametrize("rows", [0, 1, 3, 8, 40, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_are_apart_or_unaligned(rows, dtype):
    _, w, bias = make(1, 200, 300, dtype, bias=True)
    gen = torch.Generator().manual_seed(rows)
    wide = torch.randn(rows + 1, 2, 411, generator=gen).to(dtype).to(DEV)
    x = wide[:rows, 1, 7:307]  # rows 822 entries apart, an odd start
    assert rows <= 1 or not x.is_contiguous()
    got = fp8_linear(x, w, bias)
    check_linear(x, w, bias, got)
    assert torch.equal(got, fp8_linear(x.contiguous(), w, bias))
    lead = fp8_linear(x.contiguous().reshape(1, rows, 1, 300), w, bias)
    assert lead.shape == (1, rows, 1, 200) and torch.equal(lead.reshape(rows, 200), got)


@gpu
@pytest.mark.parametrize("rows", [1, 4, 30, 150])
def test_numbers_that_are_none(rows):
    """A run with an infinity or a NaN makes its row NaN, and no other; zeros stay zeros, runs of tiny numbers lose only what is below their scale."""
    x, w, _ = make(rows + 3, 300, 400, torch.bfloat16)
    x[0, 5] = float("inf")
    x[1, 399] = float("nan")
    x[2] = 0
    x[2, 130:140] = 2.0**-126
    got = fp8_linear(x, w)
    assert torch.isnan(got[:2]).all() and torch.isfinite(got[2:]).all() and got[2].abs().max() < 2.0**-90
    check_linear(x[2:], w, None, got[2:])
    layer = Fp8GatedMLP(w, Fp8Weights(w.values[:, :400], w.scales), make(1, 400, 300, torch.bfloat16)[1], "silu")
    out = layer(x)
    assert torch.isnan(out[:2]).all() and torch.isfinite(out[2:]).all()


@gpu
@pytest.mark.parametrize("rows", [1, 20, 130, 300])
def test_a_row_does_not_depend_on_the_others(rows):
    x, w, _ = make(rows, 520, 700, torch.bfloat16)
    got = fp8_linear(x, w)
    y = x.flip(0).contiguous()
    y[0] = float("nan")
    other = fp8_linear(y, w).flip(0)
    assert torch.equal(other[:-1], got[:-1]) and torch.isnan(other[-1]).all()


@gpu
@pytest.mark.parametrize("rows", [1, 24, 200])
def test_captured_and_on_two_streams(rows):
    """Two captured graphs and eager calls on two streams at once give what one call after another gives."""
    xs, w, _ = make(rows, 640, 1000, torch.bfloat16)
    layer = Fp8GatedMLP(w, w, make(1, 1000, 640, torch.bfloat16, seed=5)[1], "silu")
    inputs = [torch.roll(xs, i, 1).contiguous() for i in range(6)]
    want = [(fp8_linear(x, w), layer(x)) for x in inputs]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        x = inputs[i].clone()
        layer(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fp8_linear(x, w), layer(x)
        graphs.append((g, x, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(10):
        for (g, x, out), s, k in zip(graphs, streams, (turn % 6, (turn + 3) % 6)):
            with torch.cuda.stream(s):
                x.copy_(inputs[k])
                g.replay()
        torch.cuda.synchronize()
        for (g, x, out), k in zip(graphs, (turn % 6, (turn + 3) % 6)):
            assert torch.equal(out[0], want[k][0]) and torch.equal(out[1], want[k][1])
    got = {}
    for turn in range(6):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[turn, j] = fp8_linear(inputs[turn], w), layer(inputs[turn])
    torch.cuda.synchronize()
    for (turn, _), (a, b) in got.items():
        assert torch.equal(a, want[turn][0]) and torch.equal(b, want[turn][1])


@gpu
def test_weights_written_right_before_the_call():
    """The kernels ask for weights early: never for ones that the launch before may still be writing."""
    x, w, _ = make(2, 4096, 2048, torch.bfloat16)
    other = make(2, 4096, 2048, torch.bfloat16, seed=9)[1]
    want = [fp8_linear(x, v) for v in (w, other)]
    store = Fp8Weights(w.values.clone(), w.scales.clone())
    for turn in range(40):
        v = (w, other)[turn % 2]
        store.values.view(torch.uint8).copy_(v.values.view(torch.uint8))
        store.scales.copy_(v.scales)
        assert torch.equal(fp8_linear(x, store), want[turn % 2])
