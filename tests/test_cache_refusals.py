"""Calls of the rotary and 8-bit cache entry points that are refused, on the CPU: the HIP library checks its arguments before it asks for
a device, so nothing here runs on one."""
import ctypes as C

import numpy as np
import pytest

import cache_cases as K
from catgrad_amd import BackendPanic, _abi as A
from catgrad_amd.backend import HIP_LIBRARY
from oracle_loader import oracle_library

MEMORY = np.zeros(1 << 16, np.uint8)
AT = (MEMORY.ctypes.data + 255) // 256 * 256


@pytest.fixture(scope="module", params=["hip", "oracle"])
def lib(request):
    if request.param == "oracle":
        return oracle_library()
    import torch  # noqa: F401  (a process that uses both holds torch's HIP runtime)

    return A.bind(HIP_LIBRARY)


def batch(B=1, S=1, position=0, held=None, counts=None):
    return A.TokenBatch(B, S, position, held, counts)


def cache(**other):
    f = dict(k_codes=AT, v_codes=AT, k_scale=AT, v_scale=AT, kv_heads=1, dim=16, vdim=16, capacity=64, block=16)
    return A.Cache8(*[{**f, **other}[n] for n, _ in A.Cache8._fields_])


def rotary(**other):
    f = dict(batch=batch(), dtype=A.F32, q=AT, k=AT, q_out=AT, k_out=AT, q_pitch=0, k_pitch=0, q_out_pitch=0, k_out_pitch=0, heads=2, kv_heads=1, dim=16, rot_dims=16,
             interleaved=0, magnitude=1.0, turns=AT)
    return A.RotaryRows(*[{**f, **other}[n] for n, _ in A.RotaryRows._fields_])


def append(**other):
    f = dict(batch=batch(), dtype=A.F32, k=AT, v=AT, k_pitch=0, v_pitch=0, cache=cache())
    return A.CacheAppendRows(*[{**f, **other}[n] for n, _ in A.CacheAppendRows._fields_])


def attention(**other):
    f = dict(batch=batch(), dtype=A.F32, q=AT, out=AT, q_pitch=0, out_pitch=0, heads=2, cache=cache(), scale=1.0, window=0, workspace=AT, workspace_bytes=1 << 15)
    return A.CacheAttentionRows(*[{**f, **other}[n] for n, _ in A.CacheAttentionRows._fields_])


ROTARY = [(dict(dtype=A.U32), A.ERR_DTYPE), (dict(dtype=A.F8), A.ERR_DTYPE), (dict(dtype=99), A.ERR_DTYPE), (dict(q=None), A.ERR_ARG), (dict(q_out=None), A.ERR_ARG),
          (dict(k_out=None), A.ERR_ARG), (dict(turns=None), A.ERR_ARG), (dict(heads=0), A.ERR_ARG), (dict(kv_heads=0), A.ERR_ARG), (dict(heads=5000), A.ERR_ARG),
          (dict(dim=0), A.ERR_ARG), (dict(rot_dims=0), A.ERR_ARG), (dict(rot_dims=15), A.ERR_ARG), (dict(rot_dims=18), A.ERR_ARG), (dict(dim=5000), A.ERR_ARG),
          (dict(dim=1024, rot_dims=514), A.ERR_ARG), (dict(q_pitch=31), A.ERR_ARG), (dict(k_out_pitch=15), A.ERR_ARG)]
APPEND = [(dict(dtype=A.F8), A.ERR_DTYPE), (dict(k=None), A.ERR_ARG), (dict(v=None), A.ERR_ARG), (dict(k_pitch=3), A.ERR_ARG), (dict(v_pitch=15), A.ERR_ARG)]
CACHE = [(dict(k_codes=None), A.ERR_ARG), (dict(v_codes=None), A.ERR_ARG), (dict(k_scale=None), A.ERR_ARG), (dict(v_scale=None), A.ERR_ARG), (dict(kv_heads=0), A.ERR_ARG),
         (dict(dim=8), A.ERR_UNSUPPORTED), (dict(dim=40), A.ERR_UNSUPPORTED), (dict(dim=272), A.ERR_UNSUPPORTED), (dict(vdim=0), A.ERR_UNSUPPORTED),
         (dict(vdim=17), A.ERR_UNSUPPORTED), (dict(block=8), A.ERR_UNSUPPORTED), (dict(block=48), A.ERR_UNSUPPORTED), (dict(block=256), A.ERR_UNSUPPORTED),
         (dict(block=0), A.ERR_UNSUPPORTED), (dict(capacity=0), A.ERR_SHAPE), (dict(capacity=72), A.ERR_SHAPE)]
ATTENTION = [(dict(dtype=A.U32), A.ERR_DTYPE), (dict(q=None), A.ERR_ARG), (dict(out=None), A.ERR_ARG), (dict(heads=0), A.ERR_ARG), (dict(heads=3, cache=cache(kv_heads=2)), A.ERR_ARG),
             (dict(scale=float("nan")), A.ERR_ARG), (dict(scale=float("inf")), A.ERR_ARG), (dict(q_pitch=31), A.ERR_ARG), (dict(out_pitch=31), A.ERR_ARG)]


def names(cases):
    return [f"{i}_" + "_".join(c) for i, (c, _) in enumerate(cases)]


@pytest.mark.parametrize("other,status", ROTARY, ids=names(ROTARY))
def test_rotary(lib, other, status):
    assert lib.cg_rotary_noalloc(0, rotary(**other), None) == status


@pytest.mark.parametrize("other,status", APPEND + [(dict(cache=cache(**c)), s) for c, s in CACHE], ids=names(APPEND + CACHE))
def test_append(lib, other, status):
    assert lib.cg_cache_append_noalloc(0, append(**other), None) == status


@pytest.mark.parametrize("other,status", ATTENTION + [(dict(cache=cache(**c)), s) for c, s in CACHE], ids=names(ATTENTION + CACHE))
def test_attention(lib, other, status):
    assert lib.cg_cache_attention_noalloc(0, attention(**other), None) == status


def test_null_arguments(lib):
    n, turns, m = C.c_size_t(), (C.c_double * 8)(), C.c_float()
    assert lib.cg_rotary_noalloc(0, None, None) == A.ERR_ARG
    assert lib.cg_cache_append_noalloc(0, None, None) == A.ERR_ARG
    assert lib.cg_cache_attention_noalloc(0, None, None) == A.ERR_ARG
    assert lib.cg_cache_attention_workspace(None, n) == A.ERR_ARG
    assert lib.cg_cache_attention_workspace(attention(), None) == A.ERR_ARG
    assert lib.cg_rotation_turns(None, turns, m) == A.ERR_ARG
    assert lib.cg_rotation_turns(A.Rotation(dims=16, base=10.0), None, m) == A.ERR_ARG
    assert lib.cg_rotation_turns(A.Rotation(dims=16, base=10.0), turns, None) == A.ERR_ARG


def test_no_tokens_is_nothing_to_do(lib):
    n = C.c_size_t(7)
    for b in (batch(B=0), batch(S=0)):
        assert lib.cg_rotary_noalloc(0, rotary(batch=b, q=None, k=None), None) == A.OK
        assert lib.cg_cache_append_noalloc(0, append(batch=b, k=None), None) == A.OK
        assert lib.cg_cache_attention_noalloc(0, attention(batch=b, q=None), None) == A.OK
        assert lib.cg_cache_attention_workspace(attention(batch=b), n) == A.OK and n.value == 0


@pytest.mark.parametrize("other", [dict(dims=0), dict(dims=7), dict(dims=514), dict(base=0.0), dict(base=-3.0), dict(base=float("nan")), dict(scaling=4), dict(scaling=-1),
                                   dict(scaling=1), dict(scaling=1, factor=-2.0), dict(scaling=2, factor=2.0), dict(scaling=2, factor=2.0, low=4.0, high=1.0, original=8.0),
                                   dict(scaling=3, factor=2.0, low=1.0, high=4.0), dict(scaling=3, factor=2.0, low=1.0, high=4.0, original=8.0, base=0.5), dict(magnitude=-1.0)], ids=str)
def test_turns(lib, other):
    turns, m = (C.c_double * 512)(), C.c_float()
    assert lib.cg_rotation_turns(A.Rotation(**{**dict(dims=16, base=10000.0), **other}), turns, m) == A.ERR_ARG


@pytest.mark.parametrize("rotation", K.ROTATIONS, ids=str)
def test_turns_of_both_libraries(lib, rotation):
    turns, m = (C.c_double * (rotation["dims"] // 2))(), C.c_float()
    assert lib.cg_rotation_turns(A.Rotation(**rotation), turns, m) == A.OK
    want, wm = K.plain_turns(**rotation)
    np.testing.assert_allclose(list(turns), want, rtol=1e-13)
    assert abs(m.value - wm) <= 2.0 ** -23 * wm


# Memory that the HIP library's kernels could not use, and more than a launch takes (the oracle has no such limits).
HIP_ROTARY = [dict(q=AT + 2), dict(dtype=A.BF16, k=AT + 1), dict(turns=AT + 4), dict(q_pitch=40), dict(batch=batch(held=AT + 1)), dict(batch=batch(counts=AT + 2))]
HIP_APPEND = [dict(k=AT + 1), dict(cache=cache(k_codes=AT + 8)), dict(cache=cache(v_codes=AT + 1)), dict(cache=cache(k_scale=AT + 2)), dict(cache=cache(v_scale=AT + 1))]
HIP_ATTENTION = [dict(q=AT + 2), dict(out=AT + 1, dtype=A.F16), dict(cache=cache(v_codes=AT + 4)), dict(cache=cache(capacity=8192), workspace=None),
                 dict(cache=cache(capacity=8192), workspace_bytes=64), dict(cache=cache(capacity=8192), workspace=AT + 8)]


def test_memory_that_the_kernels_do_not_take():
    import torch  # noqa: F401

    lib = A.bind(HIP_LIBRARY)
    for o in HIP_ROTARY:
        assert lib.cg_rotary_noalloc(0, rotary(**o), None) == A.ERR_ARG, o
    for o in HIP_APPEND:
        assert lib.cg_cache_append_noalloc(0, append(**o), None) == A.ERR_ARG, o
    for o in HIP_ATTENTION:
        assert lib.cg_cache_attention_noalloc(0, attention(**o), None) == A.ERR_ARG, o
    n = C.c_size_t()
    assert lib.cg_cache_attention_workspace(attention(cache=cache(capacity=8192)), n) == A.OK and n.value > 64
    for big in (dict(batch=batch(B=1 << 25)), dict(batch=batch(B=1 << 13, S=1 << 13)), dict(batch=batch(B=1 << 40, S=1 << 40))):
        assert lib.cg_rotary_noalloc(0, rotary(**big), None) == A.ERR_UNSUPPORTED
        assert lib.cg_cache_append_noalloc(0, append(**big), None) == A.ERR_UNSUPPORTED
        assert lib.cg_cache_attention_noalloc(0, attention(**big), None) == A.ERR_UNSUPPORTED
    assert lib.cg_rotary_noalloc(0, rotary(batch=batch(position=1 << 41)), None) == A.ERR_RANGE
    assert lib.cg_cache_append_noalloc(0, append(cache=cache(capacity=1 << 31)), None) == A.ERR_SHAPE
    assert lib.cg_cache_append_noalloc(0, append(batch=batch(B=1 << 22, S=3), cache=cache(kv_heads=8)), None) == A.ERR_UNSUPPORTED
    for device in (-1, 64, 63):  # (never set up)
        assert lib.cg_rotary_noalloc(device, rotary(), None) == A.ERR_ARG
        assert lib.cg_cache_append_noalloc(device, append(), None) == A.ERR_ARG
        assert lib.cg_cache_attention_noalloc(device, attention(), None) == A.ERR_ARG
        assert "set up" in lib.cg_last_error().decode()


def refusals_of_blocks(be):
    """On tensors: refused with the reference of every argument given up, so that nothing is left behind."""
    z = lambda *s, dt=A.F32: be.zeros(s, dt)
    good = be.empty_cache(2, 2, 32, 16, 64, 16)
    rot = dict(dims=32, base=10000.0)
    used = be.pool_stats()[0]
    bad_rotary = [dict(q=z(2, 3, 64), heads=2, kv_heads=0, dim=31), dict(q=z(2, 64), heads=2, kv_heads=0, dim=32), dict(q=z(2, 3, 60), heads=2, kv_heads=0, dim=32),
                  dict(q=z(2, 3, 64), k=z(2, 2, 32), heads=2, kv_heads=1, dim=32), dict(q=z(2, 3, 64), k=z(2, 3, 64), heads=2, kv_heads=1, dim=32),
                  dict(q=z(0, 3, 64), heads=2, kv_heads=0, dim=32), dict(q=z(2, 3, 64), heads=2, kv_heads=0, dim=32, rotation=dict(dims=34, base=1.0)),
                  dict(q=z(2, 3, 64), heads=2, kv_heads=0, dim=32, rotation=dict(dims=32, base=0.0))]
    for a in bad_rotary:
        with pytest.raises(BackendPanic):
            be.block_rotary(position=0, **{**dict(rotation=rot), **a})
    k, v = z(2, 3, 64), z(2, 3, 32)
    for bad in (dict(k=z(2, 3, 32)), dict(v=z(2, 3, 16)), dict(v=z(2, 2, 32)), dict(k=z(2, 64)), dict(k=z(1, 3, 64)), dict(position=62), dict(position=2 ** 63),
                dict(cache={**good, "k_codes": z(2, 2, 64, 32)}), dict(cache={**good, "v_codes": z(2, 2, 4, 16, 8, dt=A.F8)}), dict(cache={**good, "k_scale": z(2, 2, 3)}),
                dict(cache={**good, "v_scale": z(2, 2, 4, dt=A.U32)}), dict(cache={**good, "k_codes": z(2, 64, 32, dt=A.F8)}),
                dict(cache=be.empty_cache(2, 2, 24, 16, 64, 16)), dict(cache=be.empty_cache(2, 2, 32, 16, 96, 48))):
        a = {**dict(k=k, v=v, cache=good, position=0), **bad}
        with pytest.raises(BackendPanic):
            be.block_cache_append(a["k"], a["v"], a["cache"], a["position"])
    q = z(2, 3, 128)
    for bad in (dict(q=z(2, 3, 64, 1)), dict(q=z(2, 3, 120)), dict(heads=3), dict(heads=0), dict(position=62), dict(scale=float("nan")), dict(q=z(1, 3, 128)),
                dict(cache={**good, "v_codes": z(2, 2, 4, 16, 16)})):
        a = {**dict(q=q, cache=good, heads=4, position=0, scale=1.0), **bad}
        with pytest.raises(BackendPanic):
            be.block_cache_attention(a["q"], a["cache"], heads=a["heads"], position=a["position"], scale=a["scale"])
    with pytest.raises(TypeError):
        be.block_rotary(q, heads=4, dim=32, angle=3)
    assert be.pool_stats()[0] <= used


def test_blocks(oracle):
    refusals_of_blocks(oracle)
