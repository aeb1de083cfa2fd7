"""Rotary positions and the 8-bit cache of the HIP library: every case of cache_cases.py on the caller's device memory and on tensors, then what
only a device has: streams, graphs, calls beside each other."""
import ctypes as C

import numpy as np
import pytest
import torch

import cache_cases as K
import cache_reference as R
from catgrad_amd import _abi as A
from test_cache_refusals import refusals_of_blocks

pytestmark = pytest.mark.gpu


def test_refusals(hip):
    refusals_of_blocks(hip)


@pytest.mark.parametrize("case", K.ROTARY, ids=str)
def test_rotary(hip, case):
    K.run_rotary(hip._lib, "cuda", case)


@pytest.mark.parametrize("rotation", K.ROTATIONS, ids=str)
@pytest.mark.parametrize("B,S,H,G,dim,position,view", [(2, 3, 2, 1, 128, 1000, True), (1, 1, 32, 8, 128, 0, False), (1, 700, 3, 0, 130, 131072, False)])
def test_block_rotary(hip, rotation, B, S, H, G, dim, position, view):
    K.run_block_rotary(hip, rotation, B, S, H, G, dim, position, view)


def test_block_rotary_of_one_row_for_all_tokens(hip):
    """A broadcast operand: its rows lie at no distance from each other."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 1, 2 * 64)).astype(np.float32)
    rotation = K.ROTATIONS[0]
    t = hip.broadcast(hip.from_numpy(x), (2, 5, 128))
    got, _ = hip.block_rotary(t, rotation=rotation, heads=2, kv_heads=0, dim=64, position=9)
    want, _ = hip.block_rotary(hip.from_numpy(np.ascontiguousarray(np.broadcast_to(x, (2, 5, 128)))), rotation=rotation, heads=2, kv_heads=0, dim=64, position=9)
    np.testing.assert_array_equal(hip.to_numpy(got), hip.to_numpy(want))
    y = rng.standard_normal((2, 1, 128)).astype(np.float32)
    t = hip.broadcast(hip.from_numpy(y), (2, 5, 128))
    got, _ = hip.block_rotary(t, rotation=rotation, heads=2, kv_heads=0, dim=64, position=9)
    want, _ = hip.block_rotary(hip.from_numpy(np.ascontiguousarray(np.broadcast_to(y, (2, 5, 128)))), rotation=rotation, heads=2, kv_heads=0, dim=64, position=9)
    np.testing.assert_array_equal(hip.to_numpy(got), hip.to_numpy(want))


def test_many_rotations(hip):
    """More rotations than a backend keeps the frequencies of, each twice."""
    for i in list(range(20)) * 2:
        K.run_block_rotary(hip, dict(dims=16, interleaved=i % 2, scaling=0, base=100.0 + i), 1, 2, 1, 1, 16, 50, False)


@pytest.mark.parametrize("case", K.APPEND, ids=str)
def test_append(hip, case):
    K.run_append(hip._lib, "cuda", case)


def test_append_values(hip):
    K.run_append_values(hip._lib, "cuda")


@pytest.mark.parametrize("name", list(K.ATTEND))
def test_attention(hip, name):
    K.run_attend_case(hip._lib, "cuda", name)


@pytest.mark.parametrize("S,H,block", [(1, 2, 16), (1, 3, 64), (9, 2, 16), (9, 2, 32), (20, 3, 16), (20, 3, 64), (20, 3, 128)])
def test_attention_values(hip, S, H, block):
    K.run_attend_values(hip._lib, "cuda", S, H, block)


@pytest.mark.parametrize("H,G,D,V,block,window,portions", [
    (4, 2, 32, 16, 16, 0, [5, 1, 1, 11, 1, 17]), (9, 3, 64, 64, 64, 0, [70, 1, 1, 1, 55, 1, 1]), (16, 8, 128, 128, 64, 40, [130, 1, 1, 33, 1]),
    (4, 1, 256, 96, 32, 0, [1] * 40), (8, 8, 80, 80, 128, 9, [3, 200, 1, 1])])
def test_together(hip, H, G, D, V, block, window, portions):
    K.run_blocks_together(hip, H, G, D, V, block, window, portions)


def test_shared_cache(hip):
    K.run_shared_cache(hip)


def test_blocks_give_their_memory_back(hip):
    hip.sync()
    before = hip.pool_stats()[0]
    for _ in range(3):
        K.run_blocks_together(hip, 2, 1, 32, 32, 16, 0, [9, 1, 1])
    hip.sync()
    assert hip.pool_stats()[0] == before


def test_block_append_in_place(hip):
    """A cache that its owner gives up is written where it lies: no memory is taken for it."""
    B, G, D, V, block, capacity = 1, 8, 128, 128, 64, 65536
    x = hip.from_numpy(np.ones((B, 1, G * D), np.float32))
    cache = hip.block_cache_append(x, x, hip.empty_cache(B, G, D, V, capacity, block), position=0)
    hip.sync()
    used, cached = hip.pool_stats()
    for at in range(1, 4):
        cache = hip.block_cache_append(x, x, {n: t.move() for n, t in cache.items()}, position=at)
    hip.sync()
    assert hip.pool_stats() == (used, cached)
    codes = hip.to_vec(cache["k_codes"]).reshape(G, capacity, D)
    assert (R.decode(codes[:, :4]) != 0).all() and not codes[:, 4:].any()
    # and what reads it in between sees what it held then: a widened copy that something asked for is not kept beyond the next append
    a = hip.to_numpy(hip.cast(cache["k_codes"], A.F32))
    cache = hip.block_cache_append(x, x, {n: t.move() for n, t in cache.items()}, position=4)
    b = hip.to_numpy(hip.cast(cache["k_codes"], A.F32))
    assert (a[0, :, 4] == 0).all() and (b[0, :, 4] != 0).all() and (a[0, :, :4] == b[0, :, :4]).all()


# ---- what a step's program keeps: its buffers, used again for every step ----------------------------------------------
class Step:
    """One layer's rotary positions, append and attention over buffers that stay where they are."""

    def __init__(self, lib, B, S, H, G, D, block, capacity, dtype, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.lib, self.g, self.dims = lib, g, (B, S, H, G, D, block, capacity)
        t = K.TYPES[dtype]
        self.qkv = torch.zeros(B * S, (H + 2 * G) * D, dtype=t[0], device="cuda")
        self.out = torch.zeros(B * S, H * D, dtype=t[0], device="cuda")
        self.cache = K.Cache("cuda", B, G, D, D, capacity, block, 0)
        self.held, self.counts = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.full((B,), S, dtype=torch.int32, device="cuda")
        self.turns = torch.tensor(K.plain_turns(**dict(dims=D, scaling=0, base=10000.0))[0], dtype=torch.float64, device="cuda")
        self.kind = t[1]
        self.need = C.c_size_t()
        K.check(lib, lib.cg_cache_attention_workspace(self.attention(None, 0), self.need))
        self.workspace = torch.empty(self.need.value + 16, dtype=torch.uint8, device="cuda")

    def batch(self):
        B, S = self.dims[:2]
        return A.TokenBatch(B, S, 0, self.held.data_ptr(), self.counts.data_ptr())

    def attention(self, workspace, size):
        B, S, H, G, D, block, capacity = self.dims
        return A.CacheAttentionRows(self.batch(), self.kind, self.qkv.data_ptr(), self.out.data_ptr(), self.qkv.stride(0), 0, H, self.cache.struct(), D ** -0.5, 0, workspace, size)

    def fill(self, held):
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=self.g, device="cuda"))
        self.held.fill_(held)

    def run(self, stream=None):
        B, S, H, G, D, block, capacity = self.dims
        lib, at, n = self.lib, self.qkv.data_ptr(), self.qkv.element_size()
        stream = torch.cuda.current_stream().cuda_stream if stream is None else stream
        p = self.qkv.stride(0)
        K.check(lib, lib.cg_rotary_noalloc(0, A.RotaryRows(self.batch(), self.kind, at, at + H * D * n, at, at + H * D * n, p, p, p, p, H, G, D, D, 0, 1.0, self.turns.data_ptr()), stream))
        K.check(lib, lib.cg_cache_append_noalloc(0, A.CacheAppendRows(self.batch(), self.kind, at + H * D * n, at + (H + G) * D * n, p, p, self.cache.struct()), stream))
        K.check(lib, lib.cg_cache_attention_noalloc(0, self.attention(self.workspace.data_ptr(), self.need.value), stream))
        return self.out


@pytest.mark.parametrize("dims,dtype", [((3, 1, 8, 2, 64, 64, 4096), "bf16"), ((2, 7, 6, 3, 128, 16, 1024), "f32"), ((1, 90, 4, 2, 96, 32, 2048), "f16")])
def test_graph(hip, dims, dtype):
    """A step captured once and replayed on new contents, with the program's own work between; two graphs with a workspace each."""
    steps = [Step(hip._lib, *dims, dtype, seed) for seed in (1, 1, 2, 2)]  # by pairs: replayed, and eager
    graphs = []
    side = torch.cuda.Stream()
    for s in steps[::2]:
        s.fill(0)
        s.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s.run()
        graphs.append(g)
    for s in steps:
        s.g.manual_seed(5)
        for t in (s.cache.k, s.cache.v, s.cache.ks, s.cache.vs):
            t.zero_()
    at = 0
    for _ in range(5):
        for i, g in enumerate(graphs):
            for s in steps[2 * i: 2 * i + 2]:
                s.fill(at)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(len(graphs)):
            got, want = steps[2 * i].out, steps[2 * i + 1].run()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and got.abs().max() > 0
            for n in ("k", "v", "ks", "vs"):
                assert torch.equal(getattr(steps[2 * i].cache, n), getattr(steps[2 * i + 1].cache, n))
        at += dims[1]


def test_streams_beside_each_other(hip):
    """Two steps on two streams at once, many times, and each alone: the same results."""
    dims = (2, 1, 8, 2, 128, 64, 8192)
    steps = [Step(hip._lib, *dims, "bf16", 7 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in steps]
    alone = []
    for s in steps:
        for t in (s.cache.k, s.cache.v):
            t.copy_(torch.randint(0, 120, t.shape, generator=s.g, device="cuda", dtype=torch.uint8))
        s.cache.ks.fill_(2.0 ** -6)
        s.cache.vs.fill_(2.0 ** -5)
        s.fill(8000)
        kept = s.qkv.clone()
        s.run()
        torch.cuda.synchronize()
        alone.append((kept, s.out.clone()))
    for _ in range(8):
        for s, (kept, _) in zip(steps, alone):
            s.qkv.copy_(kept)
            s.out.zero_()
        torch.cuda.synchronize()
        for s, st in zip(steps, streams):
            s.run(st.cuda_stream)
        torch.cuda.synchronize()
        for s, (_, want) in zip(steps, alone):
            assert torch.equal(s.out, want)


def test_raw_memory_and_tensors_agree(hip):
    """The same step on a caller's memory and on a backend's tensors, bit for bit."""
    dims = B, S, H, G, D, block, capacity = (2, 5, 6, 2, 64, 32, 320)
    s = Step(hip._lib, *dims, "f32", 4)
    cache = hip.empty_cache(B, G, D, D, capacity, block)
    for at in (0, 5, 10, 15):
        s.fill(at)
        x = s.qkv.cpu().numpy().reshape(B, S, -1)
        got = s.run().cpu().numpy().reshape(B, S, -1)
        q, k, v = (hip.from_numpy(np.ascontiguousarray(t)) for t in (x[..., : H * D], x[..., H * D: (H + G) * D], x[..., (H + G) * D:]))
        q, k = hip.block_rotary(q, k, rotation=dict(dims=D, base=10000.0), heads=H, kv_heads=G, dim=D, position=at)
        cache = hip.block_cache_append(k, v, {n: t.move() for n, t in cache.items()}, position=at)
        np.testing.assert_array_equal(hip.to_numpy(hip.block_cache_attention(q, cache, heads=H, position=at, scale=D ** -0.5)), got)
        np.testing.assert_array_equal(hip.to_vec(cache["k_codes"]), s.cache.k.cpu().numpy().reshape(-1))
        np.testing.assert_array_equal(hip.to_vec(cache["v_codes"]), s.cache.v.cpu().numpy().reshape(-1))


def test_position_for_all_and_null_counts(hip):
    """`position` in the place of held lengths, all tokens in the place of counts."""
    dims = (2, 3, 4, 2, 64, 16, 128)
    a, b = (Step(hip._lib, *dims, "f32", 4) for _ in range(2))
    b.batch = lambda: A.TokenBatch(2, 3, b.at, None, None)
    for at in (0, 3, 6):
        b.at = at
        a.fill(at)
        b.fill(999)
        assert torch.equal(a.run(), b.run())
        assert torch.equal(a.cache.k, b.cache.k) and torch.equal(a.cache.vs, b.cache.vs)


def test_offsets_beyond_32_bits(hip):
    """A cache of more than 2^32 bytes: its last head's positions."""
    B, G, D, block, capacity = 3, 8, 256, 128, 786432
    lib, dev = hip._lib, "cuda"
    k, v = torch.zeros(B * G * capacity * D, dtype=torch.uint8, device=dev), torch.zeros(B * G * capacity * D, dtype=torch.uint8, device=dev)
    ks, vs = (torch.full((B * G * capacity // block,), 2.0 ** -117, device=dev) for _ in range(2))
    c = A.Cache8(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), G, D, D, capacity, block)
    rng = np.random.default_rng(2)
    S, held = 3, [capacity - 3, 5, capacity - 60]
    x = [K.Rows(rng.standard_normal((B, S, G * D)), "f32", dev) for _ in range(3)]
    out = K.Rows(np.zeros((B, S, G * D)), "f32", dev)
    h, n = K.lengths(dev, held, [S] * B)
    b = A.TokenBatch(B, S, 0, h.data_ptr(), n.data_ptr())
    K.check(lib, lib.cg_cache_append_noalloc(0, A.CacheAppendRows(b, A.F32, x[0].rows.data_ptr(), x[1].rows.data_ptr(), x[0].pitch, x[1].pitch, c), K.stream_of(dev)))
    a = A.CacheAttentionRows(b, A.F32, x[2].rows.data_ptr(), out.rows.data_ptr(), x[2].pitch, out.pitch, G, c, 0.05, 0, None, 0)
    need = C.c_size_t()
    K.check(lib, lib.cg_cache_attention_workspace(a, need))
    w = torch.empty(need.value + 16, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = w.data_ptr(), need.value
    K.check(lib, lib.cg_cache_attention_noalloc(0, a, K.stream_of(dev)))
    kt, vt, q = (K.f64(t.rows).reshape(B, S, G, D) for t in x)
    got = K.f64(out.rows).reshape(B, S, G, D)
    for bb in range(B):
        for g in (0, G - 1):
            hk, hv = R.Head(256, D, block), R.Head(256, D, block)  # the last blocks alone: in front of them all codes are zero
            start = held[bb] // block * block
            hk.append(held[bb] - start, kt[bb, :, g])
            hv.append(held[bb] - start, vt[bb, :, g])
            for s in range(S):
                t = held[bb] - start + s + 1
                sc = q[bb, s, g] @ hk.x[:t].T * 0.05
                wgt = np.exp(sc)
                total = wgt.sum() + start  # (weights of one for the zeros in front)
                want = wgt @ hv.x[:t] / total
                # sums of `start` ones in 32 bits, in parts: 2^-20 of the result; and as in cache_cases.py
                terms = 0.05 * np.abs(q[bb, s, g]).max() * np.abs(hk.x[:t]).sum(-1).max()
                tol = (2 * (2.0 ** -21 * terms + 2.0 ** -20 + 2.0 ** -22) + 2.0 ** -18) * (wgt @ np.abs(hv.x[:t])) / total
                K.off_by(got[bb, s, g], want, tol, f"{bb} {g} {s}")


def test_the_current_device_is_left_as_it_was(hip):
    before = torch.cuda.current_device()
    s = Step(hip._lib, 1, 1, 2, 1, 64, 64, 64, "f32", 1)
    s.fill(0)
    s.run()
    assert torch.cuda.current_device() == before
    torch.cuda.synchronize()
