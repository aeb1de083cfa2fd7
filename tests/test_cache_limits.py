"""Calls of the 8-bit cache's entry points around what one launch takes, on the CPU: the device they name is not set up, so that a call whose sizes are
taken is refused for that."""
import pytest

from catgrad_amd import _abi as A
from catgrad_amd.backend import HIP_LIBRARY
from test_cache_refusals import append, batch, cache

NOT_SET_UP = 63


@pytest.fixture(scope="module")
def lib():
    import torch  # noqa: F401  (a process that uses both holds torch's HIP runtime)

    return A.bind(HIP_LIBRARY)


# Fewer than 2^32 threads: two blocks a head of 512, 256 or 64 threads each, for keys and for values.
@pytest.mark.parametrize("sequences,tokens,kv_heads,dim,vdim,block,status", [
    (32768, 2, 64, 128, 128, 64, A.ERR_UNSUPPORTED), (32767, 2, 64, 128, 128, 64, A.ERR_ARG), (32768, 2, 64, 16, 256, 128, A.ERR_UNSUPPORTED),
    (65535, 2, 64, 64, 64, 64, A.ERR_ARG), (65535, 2, 64, 16, 16, 16, A.ERR_ARG), (65536, 1, 63, 128, 128, 64, A.ERR_ARG), (65536, 1, 128, 128, 128, 64, A.ERR_UNSUPPORTED)])
def test_appends(lib, sequences, tokens, kv_heads, dim, vdim, block, status):
    c = cache(kv_heads=kv_heads, dim=dim, vdim=vdim, block=block, capacity=4 * block)
    assert lib.cg_cache_append_noalloc(NOT_SET_UP, append(batch=batch(B=sequences, S=tokens), cache=c), None) == status
    if status == A.ERR_ARG:
        assert "set up" in lib.cg_last_error().decode()
