"""A CTA of the few-token experts that gives up waiting for its tokens: its cluster's logits are none, so no output of the layer may look like a number.

The kernels' file is built once more with a switch by which one CTA expects more bytes of its tokens than are sent, and waits a thousand polls for them."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks
from tiny_llm_b200.mlp import FewTokenExperts, TopKRouter

from tests.test_gpu_moe_few import make

CSRC = Path(__file__).resolve().parent.parent / "tiny-llm_b200" / "csrc"
pytestmark = pytest.mark.gpu


class Starved:
    """The blocks library with the other build's entry in its place."""

    def __init__(self, lib):
        self.lib, self.whole = lib, blocks.library()
        for name in ("tlb_moe_few", "tlb_moe_few_workspace", "tlb_moe_few_tokens"):
            restype, argtypes = blocks._SIGNATURES[name]
            f = getattr(lib, name)
            f.restype, f.argtypes = restype, argtypes
            setattr(self, name, f)
        lib.tlb_few_starved_waits.restype = ctypes.c_longlong

    def __getattr__(self, name):
        return getattr(self.whole, name)


@pytest.fixture(scope="module")
def starved(tmp_path_factory):
    blocks.library()
    lib = tmp_path_factory.mktemp("starved") / "few.so"
    subprocess.run(["/usr/local/cuda/bin/nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
                    "-DTLB_FEW_STARVED", "-I", str(CSRC.parent.parent / "include"), "-o", str(lib), str(CSRC / "blocks" / "blocks_moe_few.cu"), blocks.library()._name], check=True)
    return Starved(ctypes.CDLL(str(lib)))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T", [1, 5, 30])
def test_no_output_looks_like_a_number(starved, monkeypatch, T, eight):
    D, ff, E, top = 256, 200, 24, 3
    h, router, wg, wu, wd = make(T, D, ff, E, eight, seed=21)
    layer = FewTokenExperts(TopKRouter(router, None, top), wg, wu, wd, "silu")
    want = layer(h, wide=True)
    monkeypatch.setattr(blocks, "library", lambda: starved)
    layer = FewTokenExperts(TopKRouter(router, None, top), wg, wu, wd, "silu")
    assert torch.equal(layer(h, wide=True), want)
    for cta in (0, 2, 41):  # of the cluster whose choices the second launch reads, and of another
        waits = starved.lib.tlb_few_starved_waits()
        assert starved.lib.tlb_few_starve(cta) == 0
        for wide in (True, False):
            assert torch.isnan(layer(h, wide=wide)).all()
        torch.cuda.synchronize()
        assert starved.lib.tlb_few_starved_waits() > waits
        assert starved.lib.tlb_few_starve(-1) == 0
        assert torch.equal(layer(h, wide=True), want)
