"""How many tokens a call of the experts for few tokens takes: never any at sizes whose bytes an int does not hold, and a workspace that grows with the sizes."""

from extensions_b200.tiny_llm_ext_b200 import blocks


def test_sizes_that_do_not_fit_take_no_token():
    few = blocks.moe_few_tokens
    dims = sorted({8 * 1013 * 97 * i for i in range(1, 2700)} | {2**e + d for e in range(14, 31) for d in (-8, 0, 8)} | {2**31 - 8})
    assert all(few(d, outputs, outputs, 1, 0, eight) == 0 for d in dims if 12296 <= d < 2**31 for outputs in (1, 1024) for eight in (False, True))
    assert all(few(64, 64, 64, 2, groups) == 0 for groups in (65, 2**20, 2**30, 2**31 - 1)) and few(64, 64, 64, 2, 64) == 32


def test_wider_rows_and_more_outputs_take_no_more_tokens():
    few = blocks.moe_few_tokens
    for eight in (False, True):
        by_width = [few(d, 64, 64, 6, 0, eight) for d in range(8, 14000, 8)]
        by_outputs = [few(2048, o, o, 8, 0, eight) for o in range(8, 1025)]
        assert by_width == sorted(by_width, reverse=True) and by_outputs == sorted(by_outputs, reverse=True) and by_width[0] == 32 and by_width[-1] == 0
