"""What the extension packs for the C entries of the 8-bit cache is the C structures, field by field and to their last byte: the library copies them whole."""

import ctypes
import re
from pathlib import Path

import pytest

from extensions_b200.tiny_llm_ext_b200 import blocks

HEADER = (Path(__file__).resolve().parent.parent / "include" / "tiny_llm_b200_blocks.h").read_text()
C = {"int": ctypes.c_int, "float": ctypes.c_float, "double": ctypes.c_double, "long long": ctypes.c_longlong}
CODES = {ctypes.c_void_p: "P", ctypes.c_longlong: "q", ctypes.c_double: "d", ctypes.c_float: "f", ctypes.c_int: "i"}


def structure(name):
    """The header's structure as ctypes would lay it out."""
    text = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct \{([^{}]*)\} " + name + ";", HEADER).group(1), flags=re.S)
    fields = []
    for line in filter(None, (part.strip() for part in text.split(";"))):
        kind, names = re.match(r"((?:const )?(?:void|int32_t|uint8_t|float|double|long long|int))\s*(.*)", line, flags=re.S).groups()
        for field in names.split(","):
            field = field.strip()
            fields.append((field.lstrip("* "), ctypes.c_void_p if field.startswith("*") else C[kind]))
    return type(name, (ctypes.Structure,), {"_fields_": fields})


@pytest.mark.parametrize("name,packed", [("tlb_fp8_append_call", blocks._FP8_APPEND), ("tlb_fp8_attention_call", blocks._FP8_ATTENTION)])
def test_packed_calls_are_the_c_structures(name, packed):
    c = structure(name)
    assert packed.size == ctypes.sizeof(c)
    codes = [CODES[kind] for _, kind in c._fields_]
    values = [i + 1 if code in "Pqi" else float(i + 1) for i, code in enumerate(codes)]
    read = c.from_buffer_copy(packed.pack(*values))
    assert [getattr(read, field) for field, _ in c._fields_] == values


def test_the_pages_structure_is_the_header_s():
    c = structure("tlb_fp8_pages")
    assert [f for f, _ in c._fields_] == [f for f, _ in blocks.Fp8Pages._fields_] and ctypes.sizeof(c) == ctypes.sizeof(blocks.Fp8Pages)
