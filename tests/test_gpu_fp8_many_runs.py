"""More runs of 128 than a thread's number in 32 bits holds: 2^28 rows of one run each, 16 threads a run."""

import pytest
import torch

from tiny_llm_b200.fp8 import Fp8Weights, fp8_linear

pytestmark = pytest.mark.gpu


def test_rows_behind_the_threads_of_32_bits():
    D, n, rows = 8, 8, 2**28 + 1000
    if torch.cuda.mem_get_info()[0] < 40 * 2**30:
        pytest.skip("needs 40 GB")
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = Fp8Weights.from_tensor(torch.randn(n, D, generator=gen, device="cuda"))
    piece = torch.randn(1 << 20, D, generator=gen, device="cuda").to(torch.bfloat16)
    x = piece.repeat(rows // len(piece) + 1, 1)[:rows]
    got = fp8_linear(x, w)
    want = fp8_linear(piece, w)
    for start in range(0, rows, len(piece)):
        here = got[start : start + len(piece)]
        assert torch.equal(here, want[: len(here)]), start


def test_more_rows_than_an_int_holds_are_refused():
    w = Fp8Weights.from_tensor(torch.ones(8, 8, device="cuda"))
    for rows in (2**31, 2**32 + 1):
        with pytest.raises(RuntimeError, match="rows"):
            fp8_linear(torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda").expand(rows, 8), w)  # one row of memory: refused ahead of any copy
