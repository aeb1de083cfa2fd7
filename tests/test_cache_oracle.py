"""Rotary positions and the 8-bit cache of the CPU oracle against the plain statements of cache_reference.py."""
import pytest

import cache_cases as K


@pytest.mark.parametrize("case", [c for c in K.ROTARY if c[3] * c[4] * c[6] < 40000], ids=str)
def test_rotary(oracle, case):
    K.run_rotary(oracle._lib, "cpu", case)


@pytest.mark.parametrize("rotation", K.ROTATIONS, ids=str)
def test_turns(oracle, rotation):
    K.run_turns(oracle, rotation)


@pytest.mark.parametrize("rotation", K.ROTATIONS, ids=str)
def test_block_rotary(oracle, rotation):
    K.run_block_rotary(oracle, rotation, 2, 3, 2, 1, 128, 1000, True)


@pytest.mark.parametrize("case", K.APPEND, ids=str)
def test_append(oracle, case):
    K.run_append(oracle._lib, "cpu", case)


def test_append_values(oracle):
    K.run_append_values(oracle._lib, "cpu")


@pytest.mark.parametrize("name", [n for n, c in K.ATTEND.items() if c[1] * c[9] * max(c[7]) * c[3] < 2e7 or max(c[7]) > 2 ** 31])
def test_attention(oracle, name):
    K.run_attend_case(oracle._lib, "cpu", name)


@pytest.mark.parametrize("S,H,block", [(1, 2, 16), (3, 2, 64)])
def test_attention_values(oracle, S, H, block):
    K.run_attend_values(oracle._lib, "cpu", S, H, block)


def test_together(oracle):
    K.run_blocks_together(oracle, 4, 2, 32, 16, 16, 0, [5, 1, 1, 11, 1, 17])


def test_shared_cache(oracle):
    K.run_shared_cache(oracle)
