"""The cases of cache_cases_wide.py on the HIP library."""
import ctypes as C

import numpy as np
import pytest
import torch

import cache_cases as K
import cache_cases_wide as W
from catgrad_amd import _abi as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", list(W.WIDE))
def test_attention(hip, name):
    K.run_attend_case(hip._lib, "cuda", name, cases=W.WIDE)


@pytest.mark.parametrize("case", W.VALUES, ids=str)
def test_values(hip, case):
    W.run_values(hip._lib, "cuda", *case)


@pytest.mark.parametrize("case", W.GROWING, ids=str)
def test_growing(hip, case):
    W.run_growing(hip._lib, "cuda", *case)


@pytest.mark.parametrize("dtype,S,H,D,V", [("bf16", 1, 2, 256, 256), ("bf16", 40, 2, 128, 256), ("f32", 40, 2, 96, 256), ("f16", 40, 2, 256, 128)])
def test_offsets_beyond_32_bits(hip, dtype, S, H, D, V):
    """A step of the last head of a cache of more than 2^32 bytes, its window at the end: the same step on a cache of that window's blocks."""
    lib, G, B, block, capacity, small = hip._lib, 8, 2, 128, 1536 * 1024 * 256 // min(D, V), 512
    rng = np.random.default_rng(S + D)
    q, k, v = (rng.standard_normal((S, n)) for n in (H * D, D, V))
    got = []
    for b, g, c in ((B, G, capacity), (1, 1, small)):
        bytes_of = lambda w: torch.zeros(b * g * c * w, dtype=torch.uint8, device="cuda")
        kc, vc, ks, vs = bytes_of(D), bytes_of(V), *(torch.full((b * g * c // block,), 2.0 ** -117, device="cuda") for _ in range(2))
        cache = A.Cache8(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), g, D, V, c, block)
        assert b == 1 or min(kc.numel(), vc.numel()) > 2 ** 32
        wide = lambda x, w: K.Rows(np.concatenate([np.zeros((b - 1, S, g * w)), np.concatenate([np.zeros((1, S, (g - 1) * w)), x[None]], -1)]), dtype, "cuda")
        rk, rv, rq, out = wide(k, D), wide(v, V), wide(q, H * D), K.Rows(np.zeros((b, S, g * H * V)), dtype, "cuda")
        kind = K.TYPES[dtype][1]
        for first, n in ((c - 300, S), (c - 300 + S, S)):  # the same tokens twice: a block that is begun, and one that goes on
            h, counts = K.lengths("cuda", [0] * (b - 1) + [first], [0] * (b - 1) + [n])
            batch = A.TokenBatch(b, S, 0, h.data_ptr(), counts.data_ptr())
            K.check(lib, lib.cg_cache_append_noalloc(0, A.CacheAppendRows(batch, kind, rk.rows.data_ptr(), rv.rows.data_ptr(), rk.pitch, rv.pitch, cache), K.stream_of("cuda")))
            torch.cuda.synchronize()
        a = A.CacheAttentionRows(batch, kind, rq.rows.data_ptr(), out.rows.data_ptr(), rq.pitch, out.pitch, g * H, cache, D ** -0.5, 90, None, 0)
        need = C.c_size_t()
        K.check(lib, lib.cg_cache_attention_workspace(a, need))
        w = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = w.data_ptr(), need.value
        K.check(lib, lib.cg_cache_attention_noalloc(0, a, K.stream_of("cuda")))
        torch.cuda.synchronize()
        got.append((out.rows[-1, :, -H * V:].float().cpu(), kc[-512 * D:].cpu(), vc[-512 * V:].cpu(), ks[-4:].cpu(), vs[-4:].cpu()))
        assert got[-1][0].abs().max() > 0.01
        del kc, vc
        torch.cuda.empty_cache()
    for x, y in zip(*got):
        assert torch.equal(x, y)
