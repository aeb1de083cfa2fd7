"""Sessions over the 8-bit key / value cache, on the oracle; and what a configuration may not ask for."""
import json

import numpy as np
import pytest

import session_cache_cases as cases
from catgrad_amd.runner import Session
from model_cases import TINY_LLAMA, TINY_LLAMA_UNTIED, params_of
from oracle_loader import ORACLE_LIB, oracle_library


@pytest.fixture(scope="module")
def session():
    oracle_library()
    return Session(ORACLE_LIB)


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


def test_schedules(session):
    cases.run_schedules(session, np.testing.assert_array_equal)


def test_a_step_that_fails_ends_the_request(session):
    params = params_of(TINY_LLAMA, seed=3)
    broken = dict(params)
    del broken["llama.model.norm.weight"]
    cases.load(session, TINY_LLAMA, params)
    first = session.step(1, [1, 2, 3], rows=[2])
    session.clear_params()
    for name, w in broken.items():
        session.set_param(name, w)
    with pytest.raises(Exception):
        session.step(1, [4])
    session.set_param("llama.model.norm.weight", params["llama.model.norm.weight"])
    with pytest.raises(Exception, match="earlier run"):
        session.step(1, [4])
    session.end(1)
    np.testing.assert_array_equal(session.step(1, [1, 2, 3], rows=[2]), first)
    session.end(1)


@pytest.mark.parametrize("change", [
    {"kv_cache": "f4"}, {"kv_cache": 8}, {"rope_scaling": {"rope_type": "other", "factor": 2.0}}, {"rope_scaling": {"rope_type": "linear"}},
    {"rope_scaling": {"rope_type": "llama3", "factor": 2.0}}, {"rope_scaling": {"rope_type": "linear", "factor": 0.0}},
    {"rope_scaling": {"rope_type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0, "original_max_position_embeddings": 32}},
], ids=json.dumps)
def test_configurations_that_are_refused(session, change):
    with pytest.raises(Exception):
        session.load_config({**cases.config(TINY_LLAMA), **change})


def test_architectures_without_it(session):
    with pytest.raises(Exception, match="kv_cache"):
        session.load_config({"architecture": "Loretar", "kv_cache": "f8"})


def test_heads_that_no_cache_holds(session):
    with pytest.raises(Exception, match="8-bit cache"):
        session.load_config(cases.config(TINY_LLAMA_UNTIED))


def test_no_cache_asked_for(session):
    """"f32" and no word of it answer the same, whatever the scaling says."""
    params = params_of(TINY_LLAMA, seed=3, scale=4.0)
    got = []
    for more in ({"kv_cache": "f32"}, {"kv_cache": "f32", "rope_scaling": {"rope_type": "other"}}, None):
        c = cases.config(TINY_LLAMA, **(more or {}))
        if more is None:
            del c["kv_cache"]
        session.clear_params()
        session.load_config(c)
        for name, w in params.items():
            session.set_param(name, w)
        got.append(session.step(1, [1, 2, 3], rows=[0, 1, 2], max_positions=8))
        session.end(1)
    np.testing.assert_array_equal(got[0], got[1])
    np.testing.assert_array_equal(got[0], got[2])


def test_load_pretrained(session, tmp_path):
    """The argument stands for the key of the configuration."""
    from safetensors.numpy import save_file
    params = params_of(TINY_LLAMA, seed=3, scale=4.0)
    c = cases.config(TINY_LLAMA)
    del c["kv_cache"]
    (tmp_path / "config.json").write_text(json.dumps(c))
    save_file(params, str(tmp_path / "model.safetensors"))
    got = []
    for kind in (None, "f8"):
        session.clear_params()
        session.load_pretrained(tmp_path, kv_cache=kind)
        got.append(session.step(1, [1, 2, 3], rows=[2], max_positions=8))
        session.end(1)
    cases.load(session, TINY_LLAMA, params)
    np.testing.assert_array_equal(session.step(1, [1, 2, 3], rows=[2]), got[1])
    session.end(1)
    assert not np.array_equal(got[0], got[1])


@pytest.mark.parametrize("scaling", [None, {}, {"rope_type": "default"}, {"type": "linear", "factor": 1.0}], ids=str)
def test_scaling_that_scales_nothing(session, scaling):
    params = params_of(TINY_LLAMA, seed=3, scale=4.0)
    got = []
    for more in ({}, {"rope_scaling": scaling}):
        cases.load(session, TINY_LLAMA, params, **more)
        got.append(session.step(1, range(20), rows=range(20)))
        session.end(1)
    np.testing.assert_array_equal(got[0], got[1])


def test_a_batch_is_its_sequences(session):
    """Logits of whole prompts side by side, through `forward`, are those of each alone."""
    params = params_of(TINY_LLAMA, seed=3, scale=4.0)
    cases.load(session, TINY_LLAMA, params)
    prompt = np.stack(cases.tokens_of(TINY_LLAMA, (70, 70, 70), 4))
    _, logits = session.forward(prompt)
    for b in range(3):
        np.testing.assert_array_equal(session.step(b, prompt[b], rows=range(70)), logits[b])
        session.end(b)
