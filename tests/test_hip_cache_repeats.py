"""The 8-bit cache on the HIP library: two holders of one, and calls that are made twice."""
import pytest
import torch

from cache_cases_shared import run_two_holders
from test_hip_cache import Step

pytestmark = pytest.mark.gpu


def test_two_holders(hip):
    run_two_holders(hip)


@pytest.mark.parametrize("dims,dtype", [((3, 1, 8, 2, 128, 64, 4096), "bf16"), ((2, 200, 4, 2, 128, 64, 1024), "bf16"), ((2, 200, 4, 2, 96, 16, 1024), "f32"),
                                        ((1, 1, 4, 2, 64, 64, 16384), "f32"), ((2, 200, 4, 2, 256, 32, 1024), "f16")])
def test_the_same_bits_again(hip, dims, dtype):
    """Nothing of a step depends on the order in which its workgroups run."""
    s = Step(hip._lib, *dims, dtype, 3)
    for t in (s.cache.k, s.cache.v):
        t.copy_(torch.randint(0, 120, t.shape, generator=s.g, device="cuda", dtype=torch.uint8))
    s.cache.ks.fill_(2.0 ** -6)
    s.cache.vs.copy_(2.0 ** -torch.randint(0, 12, s.cache.vs.shape, generator=s.g, device="cuda").float())
    s.fill(dims[-1] - dims[1])
    x, was, got = s.qkv.clone(), s.cache.clones(), []
    for _ in range(4):
        s.qkv.copy_(x)
        for t, w in zip((s.cache.k, s.cache.v, s.cache.ks, s.cache.vs), was):
            t.copy_(w)
        s.workspace.fill_(255)
        got.append([t.clone() for t in (s.run(), s.qkv, *s.cache.clones())])
    for g in got[1:]:
        for a, b in zip(g, got[0]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert got[0][0].isfinite().all() and got[0][0].abs().max() > 0
