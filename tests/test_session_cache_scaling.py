"""What a configuration's "rope_scaling" may say beside the numbers that sessions over the 8-bit cache follow, on the oracle."""
import json

import numpy as np
import pytest

import session_cache_cases as cases
from catgrad_amd.runner import Session
from model_cases import TINY_LLAMA, params_of
from oracle_loader import ORACLE_LIB, oracle_library


@pytest.fixture(scope="module")
def session():
    oracle_library()
    return Session(ORACLE_LIB)


@pytest.mark.parametrize("more", [{"truncate": False}, {"mscale": 0.7}, {"mscale_all_dim": 1.0}, {"mscale": 1.0, "mscale_all_dim": 1.0, "attention_factor": None}], ids=json.dumps)
def test_refused(session, more):
    with pytest.raises(Exception, match="rope_scaling"):
        session.load_config(cases.config(TINY_LLAMA, rope_scaling={**cases.SCALING["yarn"], **more}))


@pytest.mark.parametrize("more", [{"truncate": True}, {"truncate": None, "mscale": 0.0}, {"attention_factor": 0.1 * np.log(4.0) + 1.0, "mscale": 0.7}], ids=json.dumps)
def test_taken(session, more):
    params = params_of(TINY_LLAMA, seed=3, scale=4.0)
    got = []
    for m in ({}, more):
        cases.load(session, TINY_LLAMA, params, rope_scaling={**cases.SCALING["yarn"], **m})
        got.append(session.step(1, range(20), rows=range(20)))
        session.end(1)
    np.testing.assert_array_equal(got[0], got[1])
