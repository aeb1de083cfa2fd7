"""Sessions over the 8-bit key / value cache on the GPU."""
import numpy as np
import pytest

import session_cache_cases as cases
from catgrad_amd.runner import Session

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def session():
    return Session()


@pytest.mark.parametrize("name", list(cases.MODELS))
@pytest.mark.parametrize("lengths", [(9, 1, 1), (1, 1, 1), (63, 1, 1, 1), (64, 1), (5, 130, 1)], ids=str)
def test_logits_match_the_reference(session, name, lengths):
    cases.run_steps(session, name, lengths)


@pytest.mark.parametrize("scaling", [s for s in cases.SCALING if s != "none"])
def test_scaled_positions(session, scaling):
    cases.run_steps(session, "llama", (40, 1, 3), scaling)


def test_room_that_the_caller_names(session):
    cases.run_steps(session, "llama", (30, 40, 1), max_positions=71)
    cases.run_steps(session, "llama", (30, 40, 1), max_positions=32)  # named too small: it grows


def test_requests_in_turn(session):
    cases.run_interleaved(session)


@pytest.mark.parametrize("name", list(cases.MODELS))
def test_generate(session, name):
    cases.run_generate(session, name)


def test_memory_is_given_back(session):
    """Steps in place: a request's memory stays what its room needs, and goes when it ends."""
    cfg = cases.MODELS["llama"]
    params = cases.params_of(cfg, seed=3, scale=4.0)
    cases.load(session, cfg, params)
    session.step(1, [1, 2, 3], rows=[2], max_positions=256)
    session.end(1)
    session.sync()
    before = session.pool_stats()[0]
    first = session.step(1, np.arange(100) % 200, rows=[99], max_positions=256)
    session.sync()
    held = session.pool_stats()[0]
    for n in range(20):
        session.step(1, [n], rows=[0])
    session.sync()
    assert session.pool_stats()[0] == held
    session.end(1)
    session.sync()
    assert session.pool_stats()[0] == before
    np.testing.assert_array_equal(session.step(1, np.arange(100) % 200, rows=[99], max_positions=256), first)
    session.end(1)
