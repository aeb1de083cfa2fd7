"""More cases of the 8-bit cache: types and head sizes under every form of the attention, many blocks of rows and many parts, queries of extreme
sizes, and caches that grow token by token.  Tolerances: see cache_cases.py."""
import numpy as np

from cache_cases import Cache, append, run_attend, tokens_for

WIDE = {  # as ATTEND
    "96_bf16": ("bf16", 4, 2, 96, 96, 256, 64, [100, 0], [60, 33], 60, 0, 0, 0),
    "80_f16_window": ("f16", 3, 1, 80, 80, 192, 16, [20, 0], [90, 33], 90, 30, 8, 0),
    "96_16_f32": ("f32", 2, 1, 96, 16, 128, 32, [40], [70], 70, 0, 0, 0),
    "16_96_f32": ("f32", 2, 1, 16, 96, 128, 128, [50], [70], 70, 11, 3, 1),
    "80_96_bf16_skewed": ("bf16", 2, 1, 80, 96, 208, 16, [130, 3], [77, 40], 77, 0, 5, 3),
    "112_128_bf16": ("bf16", 4, 4, 112, 128, 192, 64, [80], [64], 64, 0, 0, 0),
    "128_64_f16": ("f16", 4, 4, 128, 64, 192, 64, [80], [64], 64, 0, 0, 0),
    "144_bf16": ("bf16", 2, 1, 144, 144, 192, 16, [80, 10], [50, 20], 50, 33, 1, 1),
    "256_bf16": ("bf16", 2, 1, 256, 240, 128, 128, [60], [40], 40, 0, 0, 0),
    "parts_f16": ("f16", 2, 1, 80, 80, 16384, 64, [16000], [1], 1, 0, 0, 0),
    "parts_bf16": ("bf16", 2, 1, 128, 128, 16384, 128, [16380, 900], [1, 1], 1, 0, 0, 0),
    "parts_of_portion_f32": ("f32", 2, 1, 96, 80, 6144, 32, [5900], [33], 33, 0, 0, 0),
    # more blocks of rows than a card has units, in several runs
    "many_blocks": ("f16", 16, 1, 16, 16, 256, 16, [96] * 20, [128] * 19 + [71], 128, 0, 0, 0),
    # a capacity that ends inside a tile, under rows that see all of it
    "ends_inside": ("bf16", 8, 1, 96, 128, 80, 16, [60], [20], 20, 0, 0, 0),
    "ends_inside_f32": ("f32", 8, 1, 128, 128, 144, 16, [100], [44], 44, 0, 0, 0),
}

VALUES = [("bf16", 1, 4, 128, 128, 16), ("bf16", 40, 2, 128, 128, 64), ("bf16", 40, 2, 96, 80, 16), ("bf16", 40, 2, 256, 256, 32), ("bf16", 1, 3, 256, 256, 64),
          ("f16", 40, 2, 128, 128, 32), ("f16", 5, 2, 80, 96, 16), ("f16", 40, 2, 256, 256, 64), ("f32", 40, 2, 128, 128, 16), ("f32", 40, 2, 80, 96, 32),
          ("f32", 40, 2, 256, 256, 16), ("f32", 9, 2, 128, 128, 128), ("bf16", 40, 2, 64, 64, 16)]


def run_values(lib, device, dtype, S, H, D, V, block):
    """cache_cases.run_attend_values for any type and head size, as far as the type's range goes."""
    rng = np.random.default_rng(S + block + D)
    B, T, capacity = 1, 150, 192 if block < 128 else 256
    k, v, q = tokens_for(rng, B, T, D, 0.3), tokens_for(rng, B, T, V, 0.3), rng.standard_normal((B, S, H * D))

    def case(what, k, v, q, **how):
        cache = Cache(device, B, 1, D, V, capacity, block)
        append(lib, device, cache, "f32", [0], [T], k, v)
        run_attend(lib, device, cache, dtype, [T - S], [S], q, H, what=what, **how)

    case("plain", k, v, q)
    case("scale 0", k, v, q, scale=0.0)
    case("negative scale", k, v, q, scale=-0.3)
    case("queries of zero", k, v, q * 0)
    if dtype != "f16":
        case("large queries, small keys", k * 2.0 ** -60, v, q * 2.0 ** 60)
        case("small queries, large keys", k * 2.0 ** 90, v, q * 2.0 ** -90)
        case("queries below the normal numbers", k * 2.0 ** 100, v, q * 2.0 ** -130)
    x = q.copy()
    x[:, :, ::3] *= 2.0 ** -13
    x[:, :, 1::3] *= 2.0 ** -7
    case("queries of all sizes", k, v, x)
    sharp = q.copy()
    sharp[:, :, :D] *= 40.0
    case("sharp weights", k, v, sharp)
    # (results of 16 bits in half precision hold no 2^40: there the values' sizes differ the other way)
    apart = v.copy()
    apart[:, :40] *= 2.0 ** (40 if dtype != "f16" else 8)
    apart[:, 100:120] *= 2.0 ** -40
    case("values far apart", k, apart, q)
    case("values far apart, seen in part", k, apart, q, window=60)
    for at in (0, 70, T - S, T - 1):
        x = v.copy()
        x[:, at, 3] = np.nan
        x[:, at, V - 1] = np.nan
        case(f"NaN value at {at}", k, x, q)
        case(f"NaN value at {at}, window", k, x, q, window=20)
        x = k.copy()
        x[:, at, D - 1] = np.nan
        case(f"NaN key at {at}", x, v, q)
        case(f"NaN key at {at}, window", x, v, q, window=20)
    x = apart.copy()
    x[:, 110, 1] = np.nan
    case("NaN among values far apart", k, x, q, window=30)


GROWING = [("f32", 2, 80, 112, 64, 64), ("bf16", 1, 256, 16, 256, 128), ("f16", 3, 16, 256, 64, 16), ("bf16", 2, 48, 48, 96, 32)]


def run_growing(lib, device, dtype, G, D, V, capacity, block):
    """One token after the other, each larger than the one before at first, for sequences that begin at different places."""
    rng = np.random.default_rng(D + V)
    starts = [0, 1, block - 1, block // 2 + 3, capacity - 4, capacity + 5]
    B = len(starts)
    cache = Cache(device, B, G, D, V, capacity, block)
    full = [min(s, capacity) for s in starts]
    append(lib, device, cache, dtype, [0] * B, full, tokens_for(rng, B, max(full), G * D), tokens_for(rng, B, max(full), G * V))
    held = list(starts)
    for n in range(12):
        counts = [1] * B
        counts[n % B] = 0
        size = 2.0 ** (n if n < 8 else -n)
        was = cache.clones()
        append(lib, device, cache, dtype, held, counts, size * tokens_for(rng, B, 1, G * D, 0.2), size * tokens_for(rng, B, 1, G * V, 0.2), wide=n % 3, skew=n % 2)
        held = [h + c for h, c in zip(held, counts)]
        cache.compare(held, was)
