"""How the kernels of the 8-bit cache read what the launches in front of them write: they are resident while those still run (programmatic dependent launch), so through
L2, never as memory that nobody writes or through a line that an SM may have read before."""

import re
from pathlib import Path

import pytest

BLOCKS = Path(__file__).resolve().parent.parent / "tiny-llm_b200" / "csrc" / "blocks"
FILES = ("blocks_fp8_append.cu", "blocks_fp8_attention.cuh", "blocks_fp8_attention.cu", "blocks_fp8_portion.cu")


def device_source(name):
    """Without comments, and without the C entries and the host's checks."""
    source = re.sub(r"//[^\n]*", "", (BLOCKS / name).read_text())
    for host in (r"\nint f8_check_step\(.*?\n}\n", r"\nstatic AtPlan any_plan\(.*?\n}\n"):
        source = re.sub(host, "\n", source, flags=re.S)
    return source.split('extern "C"')[0]


@pytest.mark.parametrize("name", FILES)
def test_nothing_is_read_as_memory_that_nobody_writes(name):
    assert not re.search(r"__ldg|\.nc\b|ldg_stream|__restrict__", device_source(name))


@pytest.mark.parametrize("name", FILES)
def test_lengths_tables_scales_and_pieces_are_read_through_l2(name):
    source = device_source(name)
    plain = re.findall(r"(?:\b(?:a\.|pg\.)?(?:lens|table|key_scales|value_scales|maxima|parts)\b(?:\s*\+[^;\[\]]*)?\[[^;]*?\](?!\s*=[^=])|\*scale_at\b(?!\s*=))", source)
    plain += re.findall(r"reinterpret_cast<const (?:float4|uint4) \*>\(numbers[^;]*?\)\[i\]|\b(?:x|q|from)\[(?:d|e|64 \* p \+ e)\]", source)
    # numbers of the sums' own CTA (part, js) and of its registers are none of these
    assert [p for p in plain if not p.startswith("x[e]")] == []
    reads = {"blocks_fp8_append.cu": ("a.lens", "a.table", "pg.key_scales", "pg.value_scales"), "blocks_fp8_attention.cuh": ("a.lens",),
             "blocks_fp8_attention.cu": ("table", "pg.key_scales", "pg.value_scales", "maxima", "parts"), "blocks_fp8_portion.cu": ("table", "scales", "pg.key_scales", "pg.value_scales", "from")}[name]
    for what in reads:
        assert re.search(r"ld_cg\(\s*" + re.escape(what) + r"\b", source), what
