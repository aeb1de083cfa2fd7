"""The cases of session_cache_cases_range.py on the oracle."""
import pytest

import session_cache_cases_range as cases
from catgrad_amd.runner import Session
from oracle_loader import ORACLE_LIB, oracle_library


@pytest.mark.parametrize("name", ["llama", "qwen3"])
def test_tokens_of_zeros(name):
    oracle_library()
    cases.run_tokens_of_zeros(Session(ORACLE_LIB), name)
