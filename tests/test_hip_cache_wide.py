"""The cases of cache_cases_wide.py on the HIP library."""
import pytest

import cache_cases as K
import cache_cases_wide as W

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", list(W.WIDE))
def test_attention(hip, name):
    K.run_attend_case(hip._lib, "cuda", name, cases=W.WIDE)


@pytest.mark.parametrize("case", W.VALUES, ids=str)
def test_values(hip, case):
    W.run_values(hip._lib, "cuda", *case)


@pytest.mark.parametrize("case", W.GROWING, ids=str)
def test_growing(hip, case):
    W.run_growing(hip._lib, "cuda", *case)
