"""Cases of rotary positions and the 8-bit key / value cache, run on the CPU oracle and on the HIP library against the plain statements of
cache_reference.py.

Tolerances.  A rounding is off by at most half a step, HALF[dtype] relative to the value.  Rotary: the angle's fraction of a turn has
2^-25 of a turn (2^-22.3 as an angle), cosine and sine two steps of 2^-24 each, three more roundings: below 2^-20 of the pair's size
together.  Attention: a score is off by 2^-23 of its row's largest query value times the key's values added up (the query's
pieces), as much again for the rounding of the products' sums, 2^-22 for its exponent: in all TERMS = 2^-21 of `terms` and
2^-20 (bfloat16 queries may be two codes of four bits, the second in steps of 2^-14 where the row's largest is 2^7 or more: off by
half of one, 2^-22 of the largest, so 2^-22 + 2^-23 + 2^-22 < 2^-20 of `terms`); a weight is off by that and by its own rounding (2^-22 in two pieces, 2^-11 in one), in the numerator and in the sum."""
import ctypes as C

import numpy as np
import torch

import cache_reference as R
from catgrad_amd import F16, F32, BF16, _abi as A

TYPES = {"f32": (torch.float32, F32), "f16": (torch.float16, F16), "bf16": (torch.bfloat16, BF16)}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
WEIGHT = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -11}
TERMS = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": 2.0 ** -20}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the smallest values


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def check(lib, status):
    assert status == A.OK, lib.cg_last_error().decode()


def off_by(got, want, tol, what):
    """NaN at the same places, and the rest within tol."""
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"{what}: NaN at other places"
    bad = ~nan & ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, by up to {np.max(np.where(bad, np.abs(got - want) / tol, 0)):.3g} of what is allowed"


class Rows:
    """Rows [sequences, tokens, width] in memory of a device as a caller may hold them: `wide` more elements in a row, and `skew`
    elements behind an aligned address."""

    def __init__(self, x, dtype, device, wide=0, skew=0, fill=0.0):
        B, S, W = x.shape
        self.pitch = W + wide
        self.all = torch.full((B * S * self.pitch + skew + 16,), fill, dtype=TYPES[dtype][0], device=device)
        self.rows = self.all[skew: skew + B * S * self.pitch].view(B, S, self.pitch)[..., :W]
        self.rows.copy_(torch.as_tensor(x).to(TYPES[dtype][0]))
        self.before = self.all.clone()

    def untouched(self, counts):
        """Nothing behind the rows' width, behind the counts or behind the last row has changed."""
        mine, was = self.all.clone(), self.before.clone()
        skew = self.rows.storage_offset()
        for m in (mine, was):
            v = m[skew: skew + self.rows.shape[0] * self.rows.shape[1] * self.pitch].view(self.rows.shape[0], self.rows.shape[1], self.pitch)
            for b, n in enumerate(counts):
                v[b, :n, : self.rows.shape[2]] = 0
        return bool((torch.nan_to_num(mine.float(), 9.0) == torch.nan_to_num(was.float(), 9.0)).all())


def values_of(dtype, x):
    """x as values of the type, in 64 bits."""
    return f64(torch.as_tensor(np.asarray(x)).to(TYPES[dtype][0]))


def lengths(device, held, counts):
    t = [torch.tensor(x, dtype=torch.int64, device=device).to(torch.int32) for x in (held, counts)]
    return t


def stream_of(device):
    return torch.cuda.current_stream().cuda_stream if device != "cpu" else None


# ---- rotary ----------------------------------------------------------------------------------------------------------
ROTARY = [  # dtype, held, counts, tokens, heads, kv heads, dim, turned, interleaved, in place, wide, skew
    ("f32", [0], [1], 1, 1, 1, 64, 64, False, False, 0, 0), ("f32", [131071], [1], 1, 32, 8, 64, 64, False, False, 512, 0),
    ("f32", [7, 100000, 3], [5, 2, 0], 5, 4, 2, 128, 64, True, False, 0, 0), ("f32", [4294967295], [3], 3, 3, 0, 80, 48, False, True, 16, 0),
    ("f32", [5, 9], [9, 4], 9, 3, 1, 10, 6, True, False, 3, 1), ("f32", [5, 9], [9, 4], 9, 3, 1, 7, 2, False, False, 1, 1),
    ("bf16", [0, 0, 70000, 12], [1, 1, 1, 1], 1, 16, 8, 128, 128, False, False, 0, 0), ("bf16", [30], [300], 300, 9, 3, 64, 64, True, True, 64, 0),
    ("bf16", [30, 2], [3, 7], 7, 5, 5, 96, 96, False, False, 5, 3), ("f16", [1000000], [40], 40, 8, 2, 256, 128, False, False, 8, 0),
    ("f16", [8, 8, 8], [0, 33, 12], 33, 6, 6, 80, 80, True, False, 0, 0), ("f16", [77], [6], 6, 2, 1, 512, 512, False, False, 0, 1),
    ("f32", [50], [1100], 1100, 2, 1, 64, 32, False, False, 0, 0), ("bf16", [50, 1], [2000, 1999], 2000, 1, 1, 16, 16, False, False, 0, 0)]


def run_rotary(lib, device, case, seed=0):
    dtype, held, counts, S, H, G, D, rot, inter, in_place, wide, skew = case
    rng = np.random.default_rng(seed)
    B, magnitude = len(held), 1.25
    turns = rng.uniform(0, 0.2, rot // 2) * 10.0 ** -rng.uniform(0, 5, rot // 2)
    x = [Rows(rng.standard_normal((B, S, h * D)) * 3, dtype, device, wide, skew, 5.0) for h in (H, G)]
    y = x if in_place else [Rows(np.full((B, S, h * D), -2.0), dtype, device, wide + 2, skew, 6.0) for h in (H, G)]
    want = [f64(t.rows) for t in x]
    h, c = lengths(device, held, counts)
    at = torch.tensor(turns, dtype=torch.float64, device=device)
    a = A.RotaryRows(A.TokenBatch(B, S, 0, h.data_ptr(), c.data_ptr()), TYPES[dtype][1], x[0].rows.data_ptr(), x[1].rows.data_ptr() if G else None,
                     y[0].rows.data_ptr(), y[1].rows.data_ptr() if G else None, x[0].pitch, x[1].pitch, y[0].pitch, y[1].pitch, H, G, D, rot, inter, magnitude,
                     at.data_ptr())
    check(lib, lib.cg_rotary_noalloc(0, a, stream_of(device)))
    got = [f64(t.rows) for t in y]
    for n, (g, w, heads) in enumerate(zip(got, want, (H, G))):
        for b in range(B):
            k = counts[b]
            if not heads or not k:
                continue
            z = R.rotate(w[b, :k].reshape(k, heads, D), np.arange(held[b], held[b] + k), turns, magnitude, inter)
            size = np.zeros_like(z)
            pair = w[b, :k].reshape(k, heads, D)[..., :rot] ** 2
            if inter:
                size[..., :rot] = np.repeat(pair[..., 0::2] + pair[..., 1::2], 2, -1) ** 0.5
            else:
                size[..., :rot] = np.tile(pair[..., : rot // 2] + pair[..., rot // 2:], 2) ** 0.5
            off_by(g[b, :k].reshape(z.shape), z, size * magnitude * 2.0 ** -20 + HALF[dtype] * np.abs(z) + TINY[dtype], f"rotary {case} {'qk'[n]} {b}")
        assert y[n].untouched(counts), "rotary wrote what is not its own"


ROTATIONS = [dict(dims=64, interleaved=0, scaling=A.ROTATION_PLAIN, base=500000.0), dict(dims=48, interleaved=1, scaling=A.ROTATION_LINEAR, base=10000.0, factor=4.0),
             dict(dims=64, interleaved=0, scaling=A.ROTATION_BANDS, base=500000.0, factor=32.0, low=1.0, high=4.0, original=8192.0),
             dict(dims=128, interleaved=0, scaling=A.ROTATION_RAMP, base=1000000.0, factor=4.0, low=1.0, high=32.0, original=32768.0),
             dict(dims=32, interleaved=1, scaling=A.ROTATION_RAMP, base=10000.0, factor=16.0, low=1.0, high=32.0, original=4096.0, magnitude=1.5)]


def plain_turns(dims, scaling, base, interleaved=0, factor=0.0, low=0.0, high=0.0, original=0.0, magnitude=0.0):
    f = base ** (-np.arange(0, dims, 2) / dims)
    if scaling == A.ROTATION_LINEAR:
        f = f / factor
    elif scaling == A.ROTATION_BANDS:
        wave = 2 * np.pi / f
        smooth = (original / wave - low) / (high - low)
        mixed = (1 - smooth) * f / factor + smooth * f
        f = np.where(wave < original / high, f, np.where(wave > original / low, f / factor, mixed))
    elif scaling == A.ROTATION_RAMP:
        pair = [dims * np.log(original / (t * 2 * np.pi)) / (2 * np.log(base)) for t in (high, low)]
        a, b = max(np.floor(pair[0]), 0), min(np.ceil(pair[1]), dims - 1)
        p = np.clip((np.arange(dims // 2) - a) / max(b - a, 1e-3), 0, 1)
        f = f / factor * p + f * (1 - p)
    return f / (2 * np.pi), magnitude or (0.1 * np.log(factor) + 1 if scaling == A.ROTATION_RAMP else 1.0)


def run_turns(be, rotation):
    got, m = be.rotation_turns(**rotation)
    want, wm = plain_turns(**rotation)
    np.testing.assert_allclose(got, want, rtol=1e-13)
    assert abs(m - wm) <= 2.0 ** -23 * wm


def run_block_rotary(be, rotation, B, S, H, G, dim, position, view):
    rng = np.random.default_rng(S)
    q, k = rng.standard_normal((B, S, H * dim)).astype(np.float32), rng.standard_normal((B, S, max(G, 1) * dim)).astype(np.float32)
    from block_cases import part_of_rows
    hand = (lambda x: part_of_rows(be, x)) if view else be.from_numpy
    a, b = be.block_rotary(hand(q), hand(k) if G else None, rotation=rotation, heads=H, kv_heads=G, dim=dim, position=position)
    turns, m = plain_turns(**rotation)
    for got, x, heads in ((a, q, H), (b, k, G)):
        if not heads:
            assert got is None
            continue
        z = R.rotate(x.reshape(B, S, heads, dim), np.broadcast_to(np.arange(position, position + S), (B, S)), turns, m, rotation["interleaved"])
        off_by(be.to_numpy(got).reshape(z.shape), z, 2.0 ** -20 * m * np.abs(x).max() * 1.5 + 2.0 ** -24 * np.abs(z), f"block rotary {rotation}")


# ---- the cache -------------------------------------------------------------------------------------------------------
class Cache:
    """A cache in memory of a device, its memory filled with what must not matter, and the same as cache_reference.Head."""

    def __init__(self, device, B, G, D, V, capacity, block, stale=0xFF):
        self.shape = (B, G, D, V, capacity, block)
        n = capacity // block
        self.k = torch.full((B, G, capacity, D), stale, dtype=torch.uint8, device=device)
        self.v = torch.full((B, G, n, V, block), stale, dtype=torch.uint8, device=device)
        self.ks = torch.full((B, G, n), float("nan") if stale == 0xFF else 2.0 ** 100, device=device)
        self.vs = self.ks.clone()
        self.heads = [[(R.Head(capacity, D, block), R.Head(capacity, V, block)) for _ in range(G)] for _ in range(B)]

    def struct(self):
        B, G, D, V, capacity, block = self.shape
        return A.Cache8(self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(), G, D, V, capacity, block)

    def expect(self, held, counts, k, v):
        """The reference's append of tokens k [B, S, G * D], v."""
        B, G, D, V, _, _ = self.shape
        for b in range(B):
            for g in range(G):
                self.heads[b][g][0].append(held[b], k[b, : counts[b], g * D: (g + 1) * D])
                self.heads[b][g][1].append(held[b], v[b, : counts[b], g * V: (g + 1) * V])

    def compare(self, held, was=None):
        """Codes of the positions in front of held[b] stand for the reference's values, scales are its scales; behind them (`was`: the cache's
        clones from before) nothing has changed."""
        B, G, D, V, capacity, block = self.shape
        k = R.decode(self.k.cpu().numpy()) * np.repeat(f64(self.ks), block, -1)[..., None]
        v = (R.decode(self.v.cpu().numpy()) * f64(self.vs)[..., None, None]).swapaxes(-1, -2).reshape(B, G, capacity, V)
        for b in range(B):
            n = min(held[b], capacity)
            blocks = -(-n // block)
            for g in range(G):
                for got, scale, head in ((k, self.ks, self.heads[b][g][0]), (v, self.vs, self.heads[b][g][1])):
                    np.testing.assert_array_equal(got[b, g, :n], head.x[:n])
                    np.testing.assert_array_equal(f64(scale[b, g, :blocks]), 2.0 ** head.e[:blocks])
            if was:
                assert (self.k[b, :, n:] == was[0][b, :, n:]).all()
                lie = [t[b].permute(0, 1, 3, 2).reshape(G, capacity, V) for t in (self.v, was[1])]
                assert (lie[0][:, n:] == lie[1][:, n:]).all()
                for a, o in ((self.ks, was[2]), (self.vs, was[3])):
                    assert (torch.nan_to_num(a[b, :, blocks:], -1.0) == torch.nan_to_num(o[b, :, blocks:], -1.0)).all()

    def clones(self):
        return [t.clone() for t in (self.k, self.v, self.ks, self.vs)]


def append(lib, device, cache, dtype, held, counts, k, v, wide=0, skew=0):
    """Through cg_cache_append_noalloc, and the reference's."""
    B, S = k.shape[:2]
    rk, rv = Rows(k, dtype, device, wide, skew, float("nan")), Rows(v, dtype, device, wide, skew, float("nan"))
    h, c = lengths(device, held, counts)
    a = A.CacheAppendRows(A.TokenBatch(B, S, 0, h.data_ptr(), c.data_ptr()), TYPES[dtype][1], rk.rows.data_ptr(), rv.rows.data_ptr(), rk.pitch, rv.pitch, cache.struct())
    check(lib, lib.cg_cache_append_noalloc(0, a, stream_of(device)))
    cache.expect(held, [min(n, S) for n in counts], f64(rk.rows), f64(rv.rows))


def tokens_for(rng, B, S, width, spread=1.0):
    return rng.standard_normal((B, S, width)) * np.exp(spread * rng.standard_normal((B, S, 1)))


APPEND = [  # dtype, kv heads, dim, vdim, capacity, block, appends: (held, counts, tokens) .., wide, skew
    ("f32", 1, 16, 16, 16, 16, [([0], [1], 1), ([1], [1], 1), ([2], [14], 14)], 0, 0),
    ("f32", 2, 64, 64, 128, 64, [([0, 0], [70, 3], 70), ([70, 3], [1, 1], 1), ([71, 4], [57, 30], 57)], 0, 0),
    ("f32", 3, 48, 80, 96, 32, [([0, 5, 31], [33, 0, 2], 33), ([33, 5, 33], [1, 40, 63], 70)], 3, 1),
    ("bf16", 8, 128, 128, 256, 64, [([0] * 5, [200, 1, 64, 63, 65], 200), ([200, 1, 64, 63, 65], [1] * 5, 1), ([201, 2, 65, 64, 66], [2, 3, 1, 3, 0], 3)], 128, 0),
    ("bf16", 1, 256, 192, 256, 128, [([0], [129], 129), ([129], [127], 127)], 0, 0), ("bf16", 2, 96, 16, 80, 16, [([0, 17], [80, 9], 80)], 7, 3),
    ("f16", 2, 80, 96, 304, 16, [([0], [300], 300), ([300], [4], 4)], 0, 0), ("f16", 4, 256, 256, 256, 128, [([3, 100], [253, 77], 253)], 0, 0),
    # positions behind the capacity, more tokens than there are
    ("f32", 1, 32, 32, 32, 16, [([30, 32, 4294967295, 0], [5, 5, 5, 9], 5)], 0, 0)]


def run_append(lib, device, case, seed=0):
    dtype, G, D, V, capacity, block, appends, wide, skew = case
    rng = np.random.default_rng(seed)
    B = len(appends[0][0])
    cache = Cache(device, B, G, D, V, capacity, block)
    full = [min(h, capacity) for h in appends[0][0]]
    for held, counts, S in ([([0] * B, full, max(full))] if any(full) else []) + appends:
        was = cache.clones()
        append(lib, device, cache, dtype, held, counts, tokens_for(rng, B, S, G * D), tokens_for(rng, B, S, G * V), wide, skew)
        cache.compare([min(h + min(n, S), capacity) for h, n in zip(held, counts)], was)


def run_append_values(lib, device):
    """Every sort of value: zeros, the smallest and the largest, ties between codes, infinities, NaN; scales that grow by a step and by very
    much, from blocks that hold nothing but zeros too."""
    ties = np.concatenate([(R.VALUES[:-1] + R.VALUES[1:]) / 2, R.VALUES, [448.0, 0.0]])
    rows = [np.zeros(16), np.full(16, 1e-40), ties[:16] / 64, ties[16:32], ties[100:116], ties[110:126], ties[126:142] / 4, np.full(16, 3.4e38), np.full(16, -3.4e38)]
    rows.append(np.array([np.inf, -np.inf, np.nan, 1.0] + [0.5] * 12))
    rows.append(np.array([447.99, 448.01, -448.0, 449.0] + [2.0 ** -i for i in range(12)]))
    for order in ([0, 1, 2, 3, 4, 5, 6, 10, 9, 7, 8], [7, 0, 9, 1], [9, 10], [0, 0, 3], [1, 2, 9, 10, 6]):
        cache = Cache(device, 1, 1, 16, 16, 32, 16)
        for n, r in enumerate(order):
            x = rows[r][None, None]
            append(lib, device, cache, "f32", [n], [1], x, x)
            cache.compare([n + 1])


def run_attend(lib, device, cache, dtype, held, counts, q, H, window=0, scale=None, wide=0, skew=0, workspace=None, what=""):
    """cg_cache_attention_noalloc of rows q [B, S, H * D] against the reference's cache; returns the results."""
    B, G, D, V, capacity, block = cache.shape
    S = q.shape[1]
    scale = D ** -0.5 if scale is None else scale
    rq, out = Rows(q, dtype, device, wide, skew, float("nan")), Rows(np.full((B, S, H * V), 3.0), dtype, device, wide, skew, 4.0)
    h, c = lengths(device, held, counts)
    a = A.CacheAttentionRows(A.TokenBatch(B, S, 0, h.data_ptr(), c.data_ptr()), TYPES[dtype][1], rq.rows.data_ptr(), out.rows.data_ptr(), rq.pitch, out.pitch, H,
                             cache.struct(), scale, window, None, 0)
    need = C.c_size_t()
    check(lib, lib.cg_cache_attention_workspace(a, need))
    if workspace is None:
        workspace = torch.full((need.value + 64,), 255, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), need.value
    check(lib, lib.cg_cache_attention_noalloc(0, a, stream_of(device)))
    assert (workspace[need.value:] == 255).all(), "written behind the workspace"
    real = [min(n, S) for n in counts]
    x, y, rep = f64(rq.rows).reshape(B, S, H, D), f64(out.rows).reshape(B, S, H, V), H // G
    for b in range(B):
        for s in range(real[b]):
            for g in range(G):
                k, v = cache.heads[b][g][0].x, cache.heads[b][g][1].x
                mine = slice(g * rep, (g + 1) * rep)
                want, size, terms = R.attend(x[b, s, mine], held[b] + s, k, v, scale, window)
                tol = (2 * (TERMS[dtype] * terms + 2.0 ** -20 + WEIGHT[dtype])) * size + HALF[dtype] * np.abs(want) + TINY[dtype]
                off_by(y[b, s, mine], want, tol, f"attention {what} sequence {b} token {s} head {g}")
    assert out.untouched(real), "attention wrote what is not its own"
    return out


ATTEND = {  # dtype, heads, kv heads, dim, vdim, capacity, block, held, counts, tokens, window, wide, skew
    "one_position": ("f32", 1, 1, 64, 64, 64, 64, [0], [1], 1, 0, 0, 0),
    "one_token": ("f32", 32, 8, 64, 64, 128, 64, [100], [1], 1, 0, 0, 0),
    "ragged_batch": ("bf16", 8, 2, 128, 128, 512, 64, [0, 1, 63, 64, 65, 400, 511], [1] * 7, 1, 0, 256, 0),
    "small_blocks": ("f16", 6, 3, 96, 80, 208, 16, [200, 15, 16], [1, 1, 1], 1, 0, 0, 0),
    "blocks_of_32": ("f32", 4, 4, 80, 96, 160, 32, [140, 31], [1, 1], 1, 0, 8, 0),
    "blocks_of_128": ("bf16", 4, 1, 64, 128, 384, 128, [300, 127, 128], [1, 1, 1], 1, 0, 0, 0),
    "smallest_heads": ("f32", 2, 1, 16, 16, 32, 16, [0, 30], [2, 2], 2, 0, 0, 0),
    "odd_rows": ("bf16", 5, 5, 48, 64, 96, 16, [50, 3], [3, 2], 3, 0, 3, 1),
    "largest_heads": ("f32", 4, 2, 256, 256, 320, 64, [250, 60], [1, 1], 1, 0, 0, 0),
    "wide_values": ("f16", 4, 2, 64, 256, 128, 64, [100], [3], 3, 0, 0, 0),
    "wide_keys": ("f32", 3, 1, 192, 16, 128, 64, [90], [5], 5, 0, 0, 0),
    "sixteen_rows": ("f32", 16, 1, 64, 64, 256, 64, [200], [1], 1, 0, 0, 0),
    "seventeen_rows": ("f32", 17, 1, 64, 64, 256, 64, [200, 9], [1, 1], 1, 0, 0, 0),
    "thirty_two_rows": ("bf16", 8, 1, 128, 128, 256, 64, [100, 31], [4, 3], 4, 0, 0, 0),
    "thirty_three_rows": ("f32", 3, 1, 128, 128, 256, 64, [100, 0], [11, 7], 11, 0, 0, 0),
    "few_rows_of_largest_heads": ("bf16", 8, 2, 240, 208, 192, 16, [100, 3], [6, 5], 6, 0, 0, 0),
    "prompt": ("bf16", 8, 2, 64, 64, 320, 64, [0, 0], [300, 171], 300, 0, 64, 0),
    "prompt_f32": ("f32", 4, 2, 128, 128, 192, 64, [0], [190], 190, 0, 0, 0),
    "prompt_of_largest_heads": ("f16", 2, 1, 256, 256, 128, 32, [0], [100], 100, 0, 0, 0),
    "portion": ("f32", 3, 3, 80, 64, 640, 16, [500, 77], [129, 64], 129, 0, 1, 3),
    "window_of_one": ("f32", 4, 1, 64, 64, 256, 16, [200, 0], [9, 9], 9, 1, 0, 0),
    "window": ("bf16", 4, 2, 64, 64, 512, 32, [400, 17], [90, 70], 90, 50, 0, 0),
    "window_beyond": ("f16", 2, 2, 64, 64, 128, 64, [60], [8], 8, 1000, 0, 0),
    "window_of_long": ("f32", 2, 1, 64, 64, 4096, 64, [4000, 10, 3000], [1, 1, 1], 1, 700, 0, 0),
    "cut_keys": ("f32", 2, 1, 64, 64, 8192, 64, [8000, 3, 2500], [1, 1, 1], 1, 0, 0, 0),
    "cut_keys_16": ("bf16", 8, 1, 128, 128, 4096, 16, [4000], [2], 2, 0, 0, 0),
    "cut_keys_of_portion": ("f16", 4, 1, 64, 80, 4096, 128, [3900, 100], [20, 11], 20, 0, 0, 0),
    "cut_keys_of_largest_heads": ("f32", 2, 1, 256, 256, 2560, 64, [2500], [1], 1, 0, 0, 0),
    "no_tokens_of_some": ("f32", 4, 2, 64, 64, 128, 64, [100, 50, 20], [0, 4, 9], 4, 0, 0, 0),
    "behind_the_capacity": ("f32", 2, 1, 64, 64, 64, 64, [62, 64, 70, 4294967295], [4, 1, 2, 1], 4, 0, 0, 0),
    "window_behind_the_capacity": ("f32", 2, 1, 64, 64, 64, 64, [62, 64, 70, 4294967295], [4, 1, 2, 1], 4, 6, 0, 0),
}


def run_attend_case(lib, device, name, seed=0, cases=ATTEND):
    dtype, H, G, D, V, capacity, block, held, counts, S, window, wide, skew = cases[name]
    rng = np.random.default_rng(seed + len(name))
    B = len(held)
    for stale in (0xFF, 0x7E):
        cache = Cache(device, B, G, D, V, capacity, block, stale)
        n = [min(h + min(c, S), capacity) for h, c in zip(held, counts)]
        most = max(n)
        append(lib, device, cache, dtype, [0] * B, n, tokens_for(rng, B, most, G * D, 0.3), tokens_for(rng, B, most, G * V, 1.0))
        q = tokens_for(rng, B, S, H * D, 0.5) * 1.5
        run_attend(lib, device, cache, dtype, held, counts, q, H, window, None, wide, skew, what=name)


def run_attend_values(lib, device, S, H, block):
    """Queries and caches of very different sizes, not a number and infinite ones among them: each touches the rows that see it alone."""
    rng = np.random.default_rng(S + block)
    B, D, V, capacity = 1, 64, 64, 192 if block < 128 else 256
    T = 150
    k, v, q = tokens_for(rng, B, T, D, 0.3), tokens_for(rng, B, T, V, 0.3), rng.standard_normal((B, S, H * D))

    def case(what, k, v, q, **how):
        cache = Cache(device, B, 1, D, V, capacity, block)
        append(lib, device, cache, "f32", [0], [T], k, v)
        run_attend(lib, device, cache, "f32", [T - S], [S], q, H, what=what, **how)

    case("plain", k, v, q)
    case("scale 0", k, v, q, scale=0.0)
    case("negative scale", k, v, q, scale=-0.3)
    case("queries of zero", k, v, q * 0)
    case("large queries, small keys", k * 2.0 ** -60, v, q * 2.0 ** 60)
    case("small queries, large keys", k * 2.0 ** 90, v, q * 2.0 ** -90)
    case("queries below the normal numbers", k * 2.0 ** 100, v, q * 2.0 ** -130)
    sharp = q.copy()
    sharp[:, :, :D] *= 40.0
    case("sharp weights", k, v, sharp)
    apart = v.copy()
    apart[:, :40] *= 2.0 ** 40
    apart[:, 100:120] *= 2.0 ** -40
    case("values far apart", k, apart, q)
    case("values far apart, seen in part", k, apart, q, window=60)
    for at in (0, 70, T - S, T - 1):
        x = v.copy()
        x[:, at, 3] = np.nan
        case(f"NaN value at {at}", k, x, q)
        case(f"NaN value at {at}, window", k, x, q, window=20)
        x = k.copy()
        x[:, at, 5] = np.nan
        case(f"NaN key at {at}", x, v, q)
        case(f"NaN key at {at}, window", x, v, q, window=20)
    for bad in (np.nan, np.inf, -np.inf):
        x = q.copy()
        x[:, 0, 1] = bad
        nan = q.copy()
        nan[:, 0, :D] = np.nan  # (an infinite query gives every key an infinite score or none: no weights)
        cache = Cache(device, B, 1, D, V, capacity, block)
        append(lib, device, cache, "f32", [0], [T], k, v)
        run_attend_as(lib, device, cache, x, nan, T - S, S, H)


def run_attend_as(lib, device, cache, q, like, held, S, H):
    """The results of queries q are those of `like` (which the reference is asked)."""
    B, G, D, V, capacity, block = cache.shape
    got = []
    for x in (q, like):
        rq, out = Rows(x, "f32", device), Rows(np.zeros((B, S, H * V)), "f32", device)
        h, c = lengths(device, [held], [S])
        a = A.CacheAttentionRows(A.TokenBatch(B, S, 0, h.data_ptr(), c.data_ptr()), F32, rq.rows.data_ptr(), out.rows.data_ptr(), 0, 0, H, cache.struct(), 0.1, 0, None, 0)
        need = C.c_size_t()
        check(lib, lib.cg_cache_attention_workspace(a, need))
        w = torch.empty(need.value + 1, dtype=torch.uint8, device=device)
        a.q_pitch, a.out_pitch, a.workspace, a.workspace_bytes = rq.pitch, out.pitch, w.data_ptr(), need.value
        check(lib, lib.cg_cache_attention_noalloc(0, a, stream_of(device)))
        got.append(f64(out.rows))
    np.testing.assert_array_equal(got[0], got[1])
    assert np.isnan(got[0][:, 0, :V]).all() and np.isfinite(got[0][:, 0, V:]).all()


# ---- on tensors of a backend -----------------------------------------------------------------------------------------
def run_blocks_together(be, H, G, D, V, block, window, portions, seed=0):
    """Rotary positions, append and attention as a layer's steps: a prompt in portions, then token by token, in place."""
    rng = np.random.default_rng(seed)
    B, total = 2, sum(portions)
    capacity = -(-total // block) * block
    rotation = dict(dims=D, interleaved=0, scaling=A.ROTATION_BANDS, base=500000.0, factor=8.0, low=1.0, high=4.0, original=64.0)
    turns, m = plain_turns(**rotation)
    cache = be.empty_cache(B, G, D, V, capacity, block)
    heads = [[(R.Head(capacity, D, block), R.Head(capacity, V, block)) for _ in range(G)] for _ in range(B)]
    at = 0
    for S in portions:
        q, k, v = (rng.standard_normal((B, S, n)).astype(np.float32) for n in (H * D, G * D, G * V))
        qt, kt = be.block_rotary(be.from_numpy(q), be.from_numpy(k), rotation=rotation, heads=H, kv_heads=G, dim=D, position=at)
        turned_q, turned_k = be.to_numpy(qt), be.to_numpy(kt)
        place = np.broadcast_to(np.arange(at, at + S), (B, S))
        for got, x, n in ((turned_q, q, H), (turned_k, k, G)):
            z = R.rotate(x.reshape(B, S, n, D), place, turns, m, 0)
            off_by(got.reshape(z.shape), z, 2.0 ** -20 * np.abs(x).max() * 1.5, "turned heads")
        cache = be.block_cache_append(kt, be.from_numpy(v), {n: t.move() for n, t in cache.items()}, position=at)
        out = be.to_numpy(be.block_cache_attention(qt, cache, heads=H, position=at, scale=D ** -0.5, window=window)).reshape(B, S, H, V)
        for b in range(B):
            for g in range(G):
                hk, hv = heads[b][g]
                hk.append(at, turned_k[b, :, g * D: (g + 1) * D])
                hv.append(at, v[b, :, g * V: (g + 1) * V])
                mine = slice(g * (H // G), (g + 1) * (H // G))
                for s in range(S):
                    want, size, terms = R.attend(turned_q[b, s].reshape(H, D)[mine].astype(np.float64), at + s, hk.x, hv.x, D ** -0.5, window)
                    off_by(out[b, s, mine], want, 2 * (2.0 ** -21 * terms + 2.0 ** -20 + 2.0 ** -22) * size + 2.0 ** -24 * np.abs(want), f"{at + s}")
        at += S
        codes = {n: be.to_vec(t) for n, t in cache.items()}
        k_values = R.decode(codes["k_codes"]).reshape(B, G, capacity, D)
        for b in range(B):
            for g in range(G):
                e = np.repeat(heads[b][g][0].e, block)[:at, None]
                np.testing.assert_array_equal(k_values[b, g, :at] * 2.0 ** e, heads[b][g][0].x[:at])


def run_shared_cache(be):
    """A cache that somebody else holds is copied: the other one keeps its contents."""
    rng = np.random.default_rng(3)
    B, G, D, V, block, capacity = 1, 2, 64, 32, 16, 48
    x = [(rng.standard_normal((B, n, G * D)).astype(np.float32), rng.standard_normal((B, n, G * V)).astype(np.float32)) for n in (20, 5, 5)]
    hand = lambda i: (be.from_numpy(x[i][0]), be.from_numpy(x[i][1]))
    first = be.block_cache_append(*hand(0), be.empty_cache(B, G, D, V, capacity, block), position=0)
    kept = {n: be.to_vec(t) for n, t in first.items()}
    second = be.block_cache_append(*hand(1), first, position=20)          # first is borrowed
    for n, t in first.items():
        np.testing.assert_array_equal(be.to_vec(t), kept[n])
    views = {n: be.reshape(t, t.shape) for n, t in second.items()}        # other handles of the same memory
    before = {n: be.to_vec(t) for n, t in views.items()}
    third = be.block_cache_append(*hand(2), {n: t.move() for n, t in second.items()}, position=20)
    for n, t in views.items():
        np.testing.assert_array_equal(be.to_vec(t), before[n])
    again = be.block_cache_append(*hand(2), first, position=20)
    for n in third:
        if n.endswith("scale"):
            continue
    q = be.from_numpy(rng.standard_normal((B, 1, 2 * G * D)).astype(np.float32))
    a, b = (be.to_numpy(be.block_cache_attention(q, c, heads=2 * G, position=24, scale=0.1)) for c in (views, second_of(be, x, hand, first)))
    np.testing.assert_array_equal(a, b)
    del again


def second_of(be, x, hand, first):
    return be.block_cache_append(*hand(1), first, position=20)
