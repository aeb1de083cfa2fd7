"""Attention over the 8-bit cache behind texts of millions of positions, on the HIP library."""
import ctypes as C

import pytest
import torch

import cache_cases as K
from catgrad_amd import _abi as A

pytestmark = pytest.mark.gpu


def test_long_texts_in_one_part(hip):
    """256 rows behind a text of 16 million positions, which is not cut.  Each channel's values are one in front of a place of its own and zero behind it.
    What the rows of a channel are off by in the mean: their own roundings, 2^-11 / 3^0.5 / 16, six times (2^-13.2), and those of the 2^18 sums that a total and a sum of
    weights are made of (2^-24 / 3 times the root of that, as they grow: 2^-16.6): below 2^-13 together.  Roundings of weights count for nothing beside so many."""
    T, S, D, block = 1 << 24, 1 << 16, 16, 128
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    lib, dev = hip._lib, "cuda"
    k = torch.randn(T, D, generator=g, device=dev).to(torch.float8_e4m3fn)
    q = torch.randn(S, D, generator=g, device=dev).half()
    ends = (torch.arange(D, device=dev) + 1) * (T // D)
    v = torch.arange(T, device=dev)[:, None] < ends  # [positions, channels]
    codes = (v.view(T // block, block, D).transpose(1, 2).contiguous() * 0x38).to(torch.uint8)
    ones = torch.ones(2, T // block, device=dev)
    cache = A.Cache8(k.data_ptr(), codes.data_ptr(), ones[0].data_ptr(), ones[1].data_ptr(), 1, D, D, T, block)
    out = torch.zeros(S, D, dtype=torch.float16, device=dev)
    a = A.CacheAttentionRows(A.TokenBatch(1, S, T - S, None, None), A.F16, q.data_ptr(), out.data_ptr(), 0, 0, 1, cache, D ** -0.5, 0, None, 0)
    need = C.c_size_t()
    K.check(lib, lib.cg_cache_attention_workspace(a, need))
    assert need.value == 0  # one part
    K.check(lib, lib.cg_cache_attention_noalloc(0, a, K.stream_of(dev)))
    off, at = [], torch.arange(T, device=dev)[:, None]
    for rows in torch.arange(0, S, S // 256, device=dev).split(16):
        scores = (k.double() @ q[rows].double().T * D ** -0.5).masked_fill_(at > T - S + rows, -float("inf"))
        sums = torch.exp(scores - scores.max()).view(D, 64, T // D // 64, -1).sum(2).sum(1).cumsum(0).T  # a channel's ones lie in front of a sixteenth of its own
        off.append(out[rows].double() / (sums / sums[:, -1:]) - 1)
    off = torch.cat(off).mean(0).abs()
    assert (off <= 2.0 ** -13).all(), off * 2 ** 13
