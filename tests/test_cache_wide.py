"""The cases of cache_cases_wide.py on the CPU oracle."""
import pytest

import cache_cases as K
import cache_cases_wide as W


@pytest.mark.parametrize("name", ["96_16_f32", "16_96_f32", "80_96_bf16_skewed", "144_bf16", "ends_inside"])
def test_attention(oracle, name):
    K.run_attend_case(oracle._lib, "cpu", name, cases=W.WIDE)


@pytest.mark.parametrize("case", [("bf16", 3, 2, 96, 80, 16), ("f16", 2, 1, 128, 128, 64), ("f32", 1, 2, 80, 96, 32)], ids=str)
def test_values(oracle, case):
    W.run_values(oracle._lib, "cpu", *case)


@pytest.mark.parametrize("case", W.GROWING, ids=str)
def test_growing(oracle, case):
    W.run_growing(oracle._lib, "cpu", *case)
