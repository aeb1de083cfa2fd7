"""Attention over values whose blocks' scales lie far from each other, at the edges of what a scale, a total and a sum of weights can hold.
Tolerances: see cache_cases.py."""
import ctypes as C

import numpy as np

import cache_reference as R

from cache_cases import HALF, TERMS, TYPES, WEIGHT, Cache, Rows, append, check, f64, lengths, off_by, run_attend, stream_of
from catgrad_amd import _abi as A

# Few rows are taken by four waves, a tile of 64 positions each in turn; many by waves that walk all tiles, cut into parts of four or more.
FEW, MANY = 256, 64
FORMS = {  # dtype, tokens, heads (one of keys and values), dim, vdim, positions that lie in one wave's tile or tiles before its next
    "few_f32": ("f32", 1, 2, 64, 64, FEW), "few_bf16": ("bf16", 1, 2, 128, 128, FEW), "few_f16": ("f16", 2, 3, 80, 96, FEW),
    "few_f32_of_256": ("f32", 1, 1, 256, 256, FEW), "few_bf16_20_rows": ("bf16", 10, 2, 64, 64, FEW),
    "many_f32": ("f32", 40, 1, 64, 64, MANY), "many_bf16": ("bf16", 20, 2, 128, 128, MANY), "many_f16": ("f16", 35, 1, 64, 128, MANY),
    "many_f32_of_96": ("f32", 40, 1, 96, 80, MANY), "many_bf16_of_96": ("bf16", 40, 1, 80, 96, MANY), "many_bf16_of_256": ("bf16", 40, 1, 256, 256, MANY),
}


def values_by(rng, V, sizes, each):
    """Values of `each` positions of each of the sizes, from half of it to all of it; size 0: zeros."""
    x = np.concatenate([np.full((each, 1), float(s)) for s in sizes])
    return (x * rng.uniform(0.5, 1.0, (len(x), V)))[None]


def attend_over(lib, device, form, block, v, what, q=None, k=None, **how):
    dtype, S, H, D, V, _ = FORMS[form]
    rng = np.random.default_rng(len(what))
    T = v.shape[1]
    cache = Cache(device, 1, 1, D, V, -(-T // block) * block, block)
    append(lib, device, cache, "f32", [0], [T], rng.standard_normal((1, T, D)) * 0.5 if k is None else k, v)
    return run_attend(lib, device, cache, dtype, [T - S], [S], rng.standard_normal((1, S, H * D)) * 0.5 if q is None else q, H, what=f"{what} {form} {block}", **how)


ZEROS = [[1, 0, 0], [1, 0, 0, 1], [1] + [0] * 11 + [1], [0, 0, 1, 0, 0, 0], [0] * 4, [1, 2.0 ** -100, 2.0 ** -100], [1, 2.0 ** -30, 2.0 ** -60, 2.0 ** -90, 2.0 ** -110, 1]]


def run_zeros(lib, device, form, block):
    """Values of one, then blocks of zeros or of next to nothing: a block of zeros has the smallest scale that there is."""
    rng = np.random.default_rng(block)
    V, tiles = FORMS[form][4], FORMS[form][5]
    for sizes in ZEROS:
        for each in {max(tiles, block), block}:  # from tile to tile, and within a tile
            attend_over(lib, device, form, block, values_by(rng, V, sizes * (64 // block if each < 64 else 1), each), f"{sizes} of {each}")


def run_between(lib, device, form, block):
    """A tile of blocks up to 15 exponents apart behind one whose scale is up to 15 exponents larger than theirs; the weights lie on its smallest block."""
    dtype, S, H, D, V, tiles = FORMS[form]
    rng = np.random.default_rng(block)
    top = 2.0 ** (14 if dtype == "f16" else 2)
    for near, far in ((-15, -30), (-15, -29), (-8, -20), (-1, -16), (-16, -31), (0, -15)):
        sizes = np.full(2 * tiles + 64, top)
        sizes[tiles:] = top * 2.0 ** near
        sizes[2 * tiles - block: 2 * tiles] = sizes[-block:] = top * 2.0 ** far
        v = sizes[None, :, None] * rng.uniform(0.5, 1.0, (1, len(sizes), V))
        k = rng.standard_normal((1, len(sizes), D)) * 0.1
        k[:, 2 * tiles - block: 2 * tiles] += 1.0
        attend_over(lib, device, form, block, v, f"{near} {far}", q=np.full((1, S, H * D), 100.0 / D), k=k, scale=1.0)


STALE_SCALES = [-2.0, -2.0 ** 127, -float("inf"), float("inf"), float("nan"), -0.0, -2.0 ** -140]


def run_stale_scales(lib, device, form, block):
    """What memory holds in the place of scales of blocks that nobody has begun does not matter."""
    dtype, S, H, D, V, _ = FORMS[form]
    rng = np.random.default_rng(block)
    for stale in STALE_SCALES:
        for T in (S + 1, 64 + block, 130):
            cache = Cache(device, 1, 1, D, V, 320 if block < 128 else 384, block)
            cache.ks.fill_(stale)
            cache.vs.fill_(stale)
            append(lib, device, cache, "f32", [0], [T], rng.standard_normal((1, T, D)), rng.standard_normal((1, T, V)))
            run_attend(lib, device, cache, dtype, [T - S], [S], rng.standard_normal((1, S, H * D)), H, what=f"{stale} {T} {form} {block}")


LARGE = [2.0 ** 112, 2.0 ** 119, 448 * 2.0 ** 119]


def run_large(lib, device, form, block, positions=200):
    """Values as large as a cache holds, of which an average is no larger."""
    dtype, S, H, D, V, _ = FORMS[form]
    rng = np.random.default_rng(block)
    for size in LARGE:
        for low in (1.0, -1.0, 0.5):
            v = size * (rng.uniform(low, 1.0, (1, positions, V)) if low < 1 else np.ones((1, positions, V)))
            attend_over(lib, device, form, block, v, f"{size} {low}")
            attend_over(lib, device, form, block, v, f"{size} {low} equal keys", k=np.ones((1, positions, D)))
    # the large ones in one part or wave of some
    v = np.ones((1, positions, V))
    v[:, positions // 3: positions // 2] = LARGE[-1]
    attend_over(lib, device, form, block, v, "some large")


def run_rows_apart(lib, device, form, block):
    """Rows that see nothing but values 2^135 smaller than those that others of their wave see.  A row's total is a 32-bit float in units of the
    largest scale that its wave has met, and its weights are 2^8 or more at their largest: the total's smallest step, 2^-149 of a unit, is 2^-157 of a result's,
    and may be lost once for each of the 16 instructions of a tile.  A scale is at most 2^-7 of its block's largest value."""
    dtype, S, H, D, V, _ = FORMS[form]
    rng = np.random.default_rng(block)
    small, large = 2.0 ** -60, 2.0 ** 75
    v = values_by(rng, V, [small, large], block)
    q, k, held = rng.standard_normal((1, S, H * D)) * 0.5, rng.standard_normal((1, 2 * block, D)) * 0.5, max(block - (S + 1) // 2, 0)
    cache = Cache(device, 1, 1, D, V, 2 * block, block)
    append(lib, device, cache, "f32", [0], [2 * block], k, v)
    rq, out = Rows(q, dtype, device), Rows(np.zeros((1, S, H * V)), dtype, device)
    h, c = lengths(device, [held], [S])
    a = A.CacheAttentionRows(A.TokenBatch(1, S, 0, h.data_ptr(), c.data_ptr()), TYPES[dtype][1], rq.rows.data_ptr(), out.rows.data_ptr(), rq.pitch, out.pitch, H,
                             cache.struct(), D ** -0.5, 0, None, 0)
    need = C.c_size_t()
    check(lib, lib.cg_cache_attention_workspace(a, need))
    assert need.value == 0  # (one part: so few positions are not cut)
    check(lib, lib.cg_cache_attention_noalloc(0, a, stream_of(device)))
    x, y = f64(rq.rows).reshape(S, H, D), f64(out.rows).reshape(S, H, V)
    keys, values = (t.x for t in cache.heads[0][0])
    for s in range(S):
        want, size, terms = R.attend(x[s], held + s, keys, values, D ** -0.5, 0)
        tol = 2 * (TERMS[dtype] * terms + 2.0 ** -20 + WEIGHT[dtype]) * size + HALF[dtype] * np.abs(want) + 16 * 2.0 ** -157 * 2.0 ** -7 * large
        off_by(y[s], want, tol, f"{form} {block} row {s}")


def run_large_scores(lib, device, form, block):
    """Scores far beyond 2^22, where a 32-bit float has no room for what an exponent is told from it by: keys that are the same weigh the same, and one that is
    larger than all others has all of the weight.  Weights then are equal, or one and zero: only the sums' and the results' roundings are left."""
    dtype, S, H, D, V, _ = FORMS[form]
    rng = np.random.default_rng(block)
    T = 150
    v = rng.uniform(0.5, 1.0, (1, T, V))
    for power in range(18, 61, 1) if dtype != "f16" else range(18, 31):
        for sign in (1.0, -1.0):
            size = 1.3 * 2.0 ** (power / 2)
            q, k = np.full((1, S, H * D), size / D ** 0.25), np.full((1, T, D), sign * size / D ** 0.25)
            for outlier in (False, True):
                if outlier:
                    k[:, 70] = 2.0 * np.abs(k[:, 70])
                cache = Cache(device, 1, 1, D, V, 192 if block < 128 else 256, block)
                append(lib, device, cache, "f32", [0], [T], k, v)
                rq, out = Rows(q, dtype, device), Rows(np.zeros((1, S, H * V)), dtype, device)
                h, c = lengths(device, [T - S], [S])
                a = A.CacheAttentionRows(A.TokenBatch(1, S, 0, h.data_ptr(), c.data_ptr()), TYPES[dtype][1], rq.rows.data_ptr(), out.rows.data_ptr(), rq.pitch, out.pitch, H,
                                         cache.struct(), D ** -0.5, 0, None, 0)
                need = C.c_size_t()
                check(lib, lib.cg_cache_attention_workspace(a, need))
                assert need.value == 0  # (so few positions are not cut)
                check(lib, lib.cg_cache_attention_noalloc(0, a, stream_of(device)))
                x, y = f64(rq.rows).reshape(S, H, D), f64(out.rows).reshape(S, H, V)
                keys, values = (t.x for t in cache.heads[0][0])
                for s in range(S):
                    want, size_of, _ = R.attend(x[s], T - S + s, keys, values, D ** -0.5, 0)
                    off_by(y[s], want, 2.0 ** -20 * size_of + HALF[dtype] * np.abs(want), f"2^{power} {sign} {outlier} {form} {block} row {s}")
