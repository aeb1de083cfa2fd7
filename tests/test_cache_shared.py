"""The case of cache_cases_shared.py on the CPU oracle."""
from cache_cases_shared import run_two_holders


def test_two_holders(oracle):
    run_two_holders(oracle)
