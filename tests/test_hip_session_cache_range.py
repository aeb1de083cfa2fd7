"""The cases of session_cache_cases_range.py on the GPU."""
import pytest

import session_cache_cases_range as cases
from catgrad_amd.runner import Session

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["llama", "qwen3"])
def test_tokens_of_zeros(name):
    cases.run_tokens_of_zeros(Session(), name)
