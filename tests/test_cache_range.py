"""The cases of cache_cases_range.py on the CPU oracle."""
import pytest

import cache_cases_range as E


@pytest.mark.parametrize("form,block", [("few_f32", 16), ("few_bf16_20_rows", 64)])
def test_zeros(oracle, form, block):
    E.run_zeros(oracle._lib, "cpu", form, block)


@pytest.mark.parametrize("form,block", [("few_bf16_20_rows", 16), ("few_f16", 32)])
def test_between(oracle, form, block):
    E.run_between(oracle._lib, "cpu", form, block)


@pytest.mark.parametrize("form,block", [("few_f32", 16), ("few_f16", 32)])
def test_stale_scales(oracle, form, block):
    E.run_stale_scales(oracle._lib, "cpu", form, block)


@pytest.mark.parametrize("form,block", [("few_f32", 16), ("few_bf16_20_rows", 64)])
def test_large(oracle, form, block):
    E.run_large(oracle._lib, "cpu", form, block)


@pytest.mark.parametrize("form,block", [("few_f32", 16), ("few_bf16_20_rows", 64)])
def test_rows_apart(oracle, form, block):
    E.run_rows_apart(oracle._lib, "cpu", form, block)


@pytest.mark.parametrize("form,block", [("few_f32", 16), ("few_f16", 64)])
def test_large_scores(oracle, form, block):
    E.run_large_scores(oracle._lib, "cpu", form, block)
