"""Attention over values at the edges of what scales and totals hold, on the HIP library."""
import pytest

import cache_cases_range as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("form", list(E.FORMS))
def test_zeros(hip, form, block):
    E.run_zeros(hip._lib, "cuda", form, block)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("form", list(E.FORMS))
def test_between(hip, form, block):
    E.run_between(hip._lib, "cuda", form, block)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("form", list(E.FORMS))
def test_stale_scales(hip, form, block):
    E.run_stale_scales(hip._lib, "cuda", form, block)


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("form", [f for f in E.FORMS if "_f16" not in f])
def test_large(hip, form, block):
    E.run_large(hip._lib, "cuda", form, block)


@pytest.mark.parametrize("form,positions", [("few_f32", 4000), ("few_f32", 20000), ("few_bf16", 4000), ("few_bf16", 20000), ("many_bf16", 4000), ("many_f32", 2000)])
def test_large_in_parts(hip, form, positions):
    E.run_large(hip._lib, "cuda", form, 64, positions)


@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("form", [f for f in E.FORMS if "_f16" not in f])
def test_rows_apart(hip, form, block):
    E.run_rows_apart(hip._lib, "cuda", form, block)


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("form", list(E.FORMS))
def test_large_scores(hip, form, block):
    E.run_large_scores(hip._lib, "cuda", form, block)
