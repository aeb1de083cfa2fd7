"""The operators of a key / value cache held in 8 bits, as cases that can be timed and checked.

Three operators, in the order in which a layer of a decoder runs them for B sequences of up to S new tokens each.  Sequence b
holds held[b] positions and brings counts[b] new tokens, which stand at held[b] .. held[b] + counts[b] - 1; tokens behind
counts[b] are padding, whose results are left as they were.

  rotary     turns pairs of values of every query and key head by the angle position * 2 pi * turns[i].  Pairs are (2 i, 2 i + 1)
             (interleaved) or (i, i + rot / 2), i < rot / 2; what lies behind the first `rot` values of a head goes along
             unchanged.  Results are multiplied by `magnitude` where they are turned.
  append     stores keys and values as E4M3 codes with a scale 2^e for each block of tokens and head: e is the smallest whole
             number from -117 to 119 with |x| <= 448 * 2^e for the finite values that the block has been given.  A block that
             held tokens keeps its e or grows it, and its codes are rounded anew then.  Keys lie as [B, G, C, D], values as
             [B, G, C / block, V, block].
  attend     out = softmax(scale * q . k) v over the positions of the cache up to a token's own, of which a window leaves the
             last `window`; consecutive H / G query heads share a key / value head.

`prepare` makes what a program has in hand: projections (as parts of one wider product's rows where `wide`), the step's lengths,
the cache as earlier steps left it, frequencies.  `run` is one call of one operator."""
import math

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one token of one sequence, heads of the 1B-size model, frequencies scaled for a long context: latency alone
        _rotary("rotary_token", "f32", 1, 1, 32, 8, 64, 64, False, 100000, "bands"),
        # one token each of a ragged batch in 16 bits, half of each head turned, pairs next to each other
        _rotary("rotary_batch_57", "bf16", 57, 1, 16, 8, 128, 64, True, 30000, "plain"),
        # prompts at once, heads of the 0.6B-size model, the ramp of frequencies that goes with a magnitude
        _rotary("rotary_prompts_4x2048", "f32", 4, 2048, 16, 8, 128, 128, False, 0, "ramp"),
        # a ragged portion behind long texts, an odd head size
        _rotary("rotary_ragged_7x301", "f16", 7, 301, 24, 6, 80, 48, True, 60000, "linear"),
        # one token each of a ragged batch: the append of every decode step
        _append("append_batch_64", "bf16", 64, 1, 8, 128, 128, 64, 2048, 2000),
        # prompts into an empty cache
        _append("append_prompts_4x2048", "f32", 4, 2048, 8, 64, 64, 64, 2304, 0),
        # a ragged portion into blocks that are part full, an odd head size, small blocks
        _append("append_ragged_7x301", "f16", 7, 301, 6, 80, 96, 16, 4096, 3500),
        # one token behind a short text: latency alone
        _attend("attend_token_512", "f32", 1, 1, 32, 8, 64, 64, 64, 512, 400, 0),
        # one token each of a ragged batch with long texts: the cache is read at the speed of memory
        _attend("attend_batch_32x16384", "bf16", 32, 1, 32, 8, 128, 128, 64, 16384, 16300, 0),
        # one token of one sequence behind a very long text: few heads, so the cache is cut into parts
        _attend("attend_token_131072", "f32", 1, 1, 16, 8, 128, 128, 128, 131072, 131000, 0),
        # prompts at once, as of the 0.6B-size model
        _attend("attend_prompts_4x2048", "bf16", 4, 2048, 16, 8, 128, 128, 64, 2048, 0, 0),
        # a ragged portion behind texts, with a window, an odd head size and small blocks
        _attend("attend_ragged_3x500", "f32", 3, 500, 12, 4, 96, 80, 16, 8192, 7500, 4096),
    ]


def _case(name, **c):
    return {**c, "name": name} if name else c


def _rotary(name, dtype, B, S, H, G, D, rot, interleaved, far, scaling, wide=True):
    return _case(name, op="rotary", dtype=dtype, B=B, S=S, H=H, G=G, D=D, rot=rot, interleaved=interleaved, far=far, scaling=scaling, wide=wide)


def _append(name, dtype, B, S, G, D, V, block, C, far, wide=True):
    return _case(name, op="append", dtype=dtype, B=B, S=S, G=G, D=D, V=V, block=block, C=C, far=far, wide=wide)


def _attend(name, dtype, B, S, H, G, D, V, block, C, far, window, wide=True):
    return _case(name, op="attend", dtype=dtype, B=B, S=S, H=H, G=G, D=D, V=V, block=block, C=C, far=far, window=window, wide=wide)


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dearest = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("rotary", "append", "attend")}
    while True:
        op = rng.choice(["rotary", "append", "attend", "attend"])
        dtype, wide = rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.7
        G = rng.choice([1, 2, 3, 4, 6, 8, 8, 16])
        H = G * rng.choice([1, 2, 3, 4, 4, 8])
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
        V = D if rng.random() < 0.7 else rng.choice([64, 80, 96, 128, 256])
        B = _spread(rng, 1, 64)
        S = 1 if rng.random() < 0.4 else _spread(rng, 1, 2500)
        far = 0 if rng.random() < 0.3 else _spread(rng, 1, 131072)
        block = rng.choice([16, 32, 64, 64, 128])
        C = -(-(far + S + rng.randint(0, 200)) // block) * block
        if op == "rotary":
            c = _rotary(None, dtype, B, S, H, G, D, rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)]), rng.random() < 0.5, far,
                        rng.choice(["plain", "linear", "bands", "ramp"]), wide)
        elif op == "append":
            c = _append(None, dtype, B, S, G, D, V, block, C, far, wide)
        else:
            c = _attend(None, dtype, B, S, H, G, D, V, block, C, far, 0 if rng.random() < 0.6 else _spread(rng, 1, far + S), wide)
        if H <= 64 and _cost(c) <= dearest[op] and B * G * C * (D + V) <= 1.1e9 and (op != "attend" or B * H * S * C <= 3e8):
            return c


def work(case):
    """Positions counted as `far` for every sequence; of a batch, tokens as `S` for every sequence."""
    c = case
    B, S, G, D, size = c["B"], c["S"], c["G"], c["D"], 4 if c["dtype"] == "f32" else 2
    if c["op"] == "rotary":
        n = B * S * (c["H"] + G)
        return {"bytes": 2 * n * D * size, "flops": 6 * n * c["rot"] / 2}
    if c["op"] == "append":
        n = B * S * G * (D + c["V"])
        return {"bytes": n * (size + 1), "flops": 2 * n}
    H, V, far, window = c["H"], c["V"], c["far"], c["window"]
    seen = sum(min(far + s + 1, window or far + s + 1) for s in range(S))  # keys of one sequence's tokens, added up
    read = min(far + S, (window + S - 1) if window else far + S)
    return {"bytes": B * (S * H * (D + V) * size + G * read * (D + V)), "flops": 2 * B * H * seen * (D + V)}


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 4e13


# ------------------------------------------------------------------------------------------------ inputs

def _turns(case):
    """Turns (of 2 pi) a position for each pair, and the magnitude that goes with them."""
    half, base, factor, original = case["rot"] // 2, 500000.0, 8.0, 8192
    f = [base ** (-i / half) for i in range(half)]
    magnitude = 1.0
    if case["scaling"] == "linear":
        f = [x / factor for x in f]
    elif case["scaling"] == "bands":  # long waves are stretched, short ones not, those between by part
        low, high = 1.0, 4.0
        part = [min(max((original * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        f = [x * (p + (1 - p) / factor) for x, p in zip(f, part)]
    elif case["scaling"] == "ramp":  # the same over the pairs' numbers
        at = [case["rot"] * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), case["rot"] - 1)
        part = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(half)]
        f = [x * (1 - p + p / factor) for x, p in zip(f, part)]
        magnitude = 0.1 * math.log(factor) + 1
    return [x / (2 * math.pi) for x in f], magnitude


def _part(g, rows, widths, dtype, wide):
    """Arrays of `rows` tokens, as parts of one wider product's rows where `wide`."""
    if not wide:
        return [torch.randn(rows, w, generator=g, device="cuda").to(dtype) for w in widths]
    return list(torch.randn(rows, sum(widths), generator=g, device="cuda").to(dtype).split(widths, 1))


_powers = []


def _power(e):
    """2^e in 64 bits, from a table: e from -150 to 150."""
    if not _powers:
        _powers.append(torch.tensor([2.0 ** i for i in range(-150, 151)], dtype=torch.float64, device="cuda"))
    return _powers[0][e.long() + 150]


def _coded(x, axes):
    """(codes as bytes, 2^e) for values x in 32 bits, one e over `axes`."""
    m, e = torch.frexp(x.abs().amax(axes, keepdim=True))
    two = _power((e - 9 + (m > 0.875).int()).clamp(-117, 119))
    return (x.double() / two).float().to(F8).view(torch.uint8), two.float()


def _cache(g, c):
    """Codes and scales of a cache that earlier steps have filled, whose heads' channels are of different sizes."""
    B, G, C, D, V, n = c["B"], c["G"], c["C"], c["D"], c["V"], c["block"]
    s = {"k_codes": torch.empty(B, G, C, D, dtype=torch.uint8, device="cuda"), "v_codes": torch.empty(B, G, C // n, V, n, dtype=torch.uint8, device="cuda"),
         "k_scale": torch.empty(B, G, C // n, device="cuda"), "v_scale": torch.empty(B, G, C // n, device="cuda")}
    channels = 0.5 + 2 * torch.rand(G, 1, 1, D, generator=g, device="cuda") ** 4
    for b in range(B):
        codes, two = _coded(torch.randn(G, C // n, n, D, generator=g, device="cuda") * channels, (2, 3))
        s["k_codes"][b], s["k_scale"][b] = codes.view(G, C, D), two.view(G, C // n)
        codes, two = _coded(torch.randn(G, C // n, V, n, generator=g, device="cuda") * 0.5, (2, 3))
        s["v_codes"][b], s["v_scale"][b] = codes, two.view(G, C // n)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, B, S, dtype = case, case["B"], case["S"], TYPES[case["dtype"]]
    # texts of different lengths, portions of different lengths; every batch has a sequence with the most of both
    held = (c["far"] * (1 - 0.5 * torch.rand(B, generator=g, device="cuda") ** 2)).long()
    counts = (S * (1 - 0.5 * torch.rand(B, generator=g, device="cuda") ** 3)).ceil().long()
    held[-1], counts[0] = c["far"], S
    s = {"case": c, "held": held.int(), "counts": counts.int()}
    if c["op"] == "rotary":
        s["q"], s["k"] = _part(g, B * S, [c["H"] * c["D"], c["G"] * c["D"]], dtype, c["wide"])
        turns, s["magnitude"] = _turns(c)
        s["turns"] = torch.tensor(turns, dtype=torch.float64, device="cuda")
        s["q_out"], s["k_out"] = torch.zeros(B * S, c["H"] * c["D"], dtype=dtype, device="cuda"), torch.zeros(B * S, c["G"] * c["D"], dtype=dtype, device="cuda")
        return s
    s.update(_cache(g, c))
    if c["op"] == "append":
        s["k"], s["v"] = _part(g, B * S, [c["G"] * c["D"], c["G"] * c["V"]], dtype, c["wide"])
        s["k"] *= 1.3  # (new tokens beyond what a block's scale takes: some grow)
    else:
        s["q"] = _part(g, B * S, [c["H"] * c["D"], 2 * c["G"] * c["D"] if c["wide"] else 1], dtype, c["wide"])[0]
        s["out"] = torch.zeros(B * S, c["H"] * c["V"], dtype=dtype, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "attend": _own_attend}[op](s)
    return {"rotary": _rotate, "append": _store, "attend": _attention}[op](s)


def _real(s):
    """[B, S, 1]: which tokens are no padding."""
    return (torch.arange(s["case"]["S"], device="cuda") < s["counts"][:, None])[:, :, None]


def _rotate(s):
    c, n = s["case"], s["case"]["rot"]
    B, S, D = c["B"], c["S"], c["D"]
    position = s["held"][:, None] + torch.arange(S, device="cuda")
    angle = (position[:, :, None].double() * (s["turns"] * (2 * math.pi)))[:, :, None, :]
    cos, sin = angle.cos().float() * s["magnitude"], angle.sin().float() * s["magnitude"]
    real = _real(s)[..., None]

    def turned(x, heads, out):
        x = x.float().view(B, S, heads, D)
        if c["interleaved"]:
            a, b = x[..., 0:n:2], x[..., 1:n:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., : n // 2], x[..., n // 2: n]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.where(real, torch.cat([r, x[..., n:]], -1).to(out.dtype), out.view(B, S, heads, D)).view(B * S, heads * D)

    return {"q": turned(s["q"], c["H"], s["q_out"]), "k": turned(s["k"], c["G"], s["k_out"])}


def _store(s):
    c = s["case"]
    B, S, G, C, n = c["B"], c["S"], c["G"], c["C"], c["block"]
    blocks = min(C // n, (S + n - 2) // n + 1)  # as many as S tokens can touch
    first = (s["held"].long() // n).clamp(max=C // n - blocks)
    at = first[:, None] + torch.arange(blocks, device="cuda")             # [B, blocks]
    place = at[:, :, None] * n + torch.arange(n, device="cuda")           # [B, blocks, n]
    token = place - s["held"][:, None, None]
    new = (token >= 0) & (token < s["counts"][:, None, None])
    old = (token < 0)
    touched = new.any(-1)                                                 # [B, blocks]
    used = old.any(-1)
    row = torch.arange(B, device="cuda")[:, None]

    def stored(x, codes, scale, width, lies_by_token):
        x = x.float().view(B, S, G, width)
        x = x[row[:, :, None], token.clamp(0, S - 1)].permute(0, 1, 3, 2, 4)               # [B, blocks, G, n, width]
        before = (codes.view(B, G, C // n, n, width) if lies_by_token else codes)[row, :, at]  # [B, blocks, G, ..]
        if not lies_by_token:
            before = before.transpose(-1, -2)
        here, past = new[:, :, None, :, None], old[:, :, None, :, None]
        size = torch.where(here & x.isfinite(), x.abs(), 0.0).amax((-1, -2), keepdim=True)
        m, e = torch.frexp(size)
        e = (e - 9 + (m > 0.875).int()).clamp(-117, 119)
        e = torch.where(size > 0, e, -117)
        had = torch.frexp(scale.transpose(1, 2)[row, at])[1][..., None, None] - 1
        e = torch.where(used[:, :, None, None, None], torch.maximum(e, had), e)
        two = _power(e)
        kept = before.contiguous().view(F8).float().double() * _power(had.clamp(-117, 119))
        value = torch.where(here, x.double(), kept) / two
        after = value.clamp(-448, 448).float().to(F8).view(torch.uint8)
        after = torch.where((here | past) & touched[:, :, None, None, None], after, before)
        if not lies_by_token:
            after = after.transpose(-1, -2)
        (codes.view(B, G, C // n, n, width) if lies_by_token else codes)[row, :, at] = after
        now = torch.where(touched[:, :, None], two[..., 0, 0].float(), scale.transpose(1, 2)[row, at])
        scale.transpose(1, 2)[row, at] = now
        return codes.view(F8), scale

    k, ks = stored(s["k"], s["k_codes"], s["k_scale"], c["D"], True)
    v, vs = stored(s["v"], s["v_codes"], s["v_scale"], c["V"], False)
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _attention(s):
    c = s["case"]
    B, S, H, G, D, V, C, n = c["B"], c["S"], c["H"], c["G"], c["D"], c["V"], c["C"], c["block"]
    k = (s["k_codes"].view(F8).float().view(B, G, C // n, n, D) * s["k_scale"][..., None, None]).view(B, G, C, D)
    v = (s["v_codes"].view(F8).float() * s["v_scale"][..., None, None]).transpose(-1, -2).reshape(B, G, C, V)
    q = s["q"].float().view(B, S, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, S * (H // G), D)
    w = torch.matmul(q, k.transpose(-1, -2)).view(B, G, S, H // G, C).mul_(D ** -0.5)
    last = s["held"][:, None] + torch.arange(S, device="cuda")
    j = torch.arange(C, device="cuda")
    hidden = j > last[..., None]
    if c["window"]:
        hidden |= j <= last[..., None] - c["window"]
    w.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    w = (w - w.amax(-1, keepdim=True)).exp_()
    sums = w.sum(-1)[..., None]
    out = torch.matmul(w.view(B, G, S * (H // G), C), v).view(B, G, S, H // G, V) / sums
    out = out.permute(0, 2, 1, 3, 4).reshape(B, S, H * V).to(s["out"].dtype)
    return torch.where(_real(s), out, s["out"].view(B, S, H * V)).view(B * S, H * V)


# ------------------------------------------------------------------------------------------------ the framework's calls

_library = []


def _lib():
    """The library, set up for calls that allocate nothing, and its argument types."""
    if not _library:
        from catgrad_amd import _abi as A
        from catgrad_amd.backend import load_hip_library

        lib = load_hip_library()
        assert lib.cg_noalloc_setup(0) == A.OK, lib.cg_last_error()
        _library[:] = [lib, A, {"f32": A.F32, "f16": A.F16, "bf16": A.BF16}]
    return _library


def _batch(A, s):
    c = s["case"]
    return A.TokenBatch(c["B"], c["S"], 0, s["held"].data_ptr(), s["counts"].data_ptr())


def _cache8(A, s):
    c = s["case"]
    return A.Cache8(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scale"].data_ptr(), s["v_scale"].data_ptr(), c["G"], c["D"], c["V"], c["C"], c["block"])


def _checked(lib, status):
    if status:
        raise RuntimeError(lib.cg_last_error().decode())


def _own_rotary(s):
    lib, A, types = _lib()
    c = s["case"]
    a = A.RotaryRows(_batch(A, s), types[c["dtype"]], s["q"].data_ptr(), s["k"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(),
                     s["q"].stride(0), s["k"].stride(0), 0, 0, c["H"], c["G"], c["D"], c["rot"], c["interleaved"], s["magnitude"], s["turns"].data_ptr())
    _checked(lib, lib.cg_rotary_noalloc(0, a, torch.cuda.current_stream().cuda_stream))
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_append(s):
    lib, A, types = _lib()
    c = s["case"]
    a = A.CacheAppendRows(_batch(A, s), types[c["dtype"]], s["k"].data_ptr(), s["v"].data_ptr(), s["k"].stride(0), s["v"].stride(0), _cache8(A, s))
    _checked(lib, lib.cg_cache_append_noalloc(0, a, torch.cuda.current_stream().cuda_stream))
    return {"k": s["k_codes"].view(F8), "v": s["v_codes"].view(F8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _own_attend(s):
    lib, A, types = _lib()
    c = s["case"]
    a = A.CacheAttentionRows(_batch(A, s), types[c["dtype"]], s["q"].data_ptr(), s["out"].data_ptr(), s["q"].stride(0), 0, c["H"], _cache8(A, s),
                             c["D"] ** -0.5, c["window"], 0, 0)
    if "workspace" not in s:  # kept with the step's buffers
        need = A.C.c_size_t()
        _checked(lib, lib.cg_cache_attention_workspace(a, need))
        s["workspace"] = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    _checked(lib, lib.cg_cache_attention_noalloc(0, a, torch.cuda.current_stream().cuda_stream))
    return s["out"]


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)


def _exact_rotary(s):
    """Turned as complex numbers, a sequence at a time."""
    c, n, D = s["case"], s["case"]["rot"], s["case"]["D"]
    out = {}
    for name, heads in (("q", c["H"]), ("k", c["G"])):
        y = torch.zeros(c["B"], c["S"], heads, D, dtype=torch.float64, device="cuda")
        for b, (held, count) in enumerate(zip(s["held"].tolist(), s["counts"].tolist())):
            x = s[name].view(c["B"], c["S"], heads, D)[b, :count].double()
            turn = torch.outer(torch.arange(held, held + count, dtype=torch.float64, device="cuda"), s["turns"])
            z = torch.polar(torch.full_like(turn, s["magnitude"]), 2 * math.pi * (turn - turn.round()))[:, None]
            head = x[..., :n].unflatten(-1, (n // 2, 2) if c["interleaved"] else (2, n // 2))
            if not c["interleaved"]:
                head = head.transpose(-1, -2)
            t = torch.view_as_real(torch.view_as_complex(head.contiguous()) * z)
            y[b, :count, :, :n] = (t if c["interleaved"] else t.transpose(-1, -2)).flatten(-2)
            y[b, :count, :, n:] = x[..., n:]
        out[name] = y.view(c["B"] * c["S"], heads * D)
    return out


def _values(codes):
    """What E4M3 bytes stand for."""
    table = np.array([(1 - 2 * (b >> 7)) * ((b & 7) / 512 if b >> 3 & 15 == 0 else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10)) for b in range(256)])
    table[[127, 255]] = np.nan
    return torch.from_numpy(table).cuda()[codes.int()]


def _two(e):
    """2^e in 64 bits, by its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest(x):
    """x rounded to the nearest value of E4M3 (ties to even), up to 448."""
    unit = _two(torch.frexp(x)[1].clamp(min=-5) - 4)
    return (torch.round(x / unit) * unit).clamp(-448, 448)


def _exact_append(s):
    c, n = s["case"], s["case"]["block"]
    B, S, G, C = c["B"], c["S"], c["G"], c["C"]
    out = {}
    for name, width in (("k", c["D"]), ("v", c["V"])):
        lies = s[name + "_codes"].view(B, G, C // n, n, width) if name == "k" else s[name + "_codes"].transpose(-1, -2)
        codes, scale = _values(lies), s[name + "_scale"].double()
        x = s[name].view(B, S, G, width).double()
        for b, (held, count) in enumerate(zip(s["held"].tolist(), s["counts"].tolist())):
            for j in range(held // n, (held + count - 1) // n + 1):
                past, t0, t1 = max(held - j * n, 0), max(j * n - held, 0), min((j + 1) * n - held, count)
                y = x[b, t0:t1].transpose(0, 1)
                m, e = torch.frexp(y.abs().amax((1, 2)) / 448)
                two = _two((e - (m == 0.5).int()).clamp(-117, 119)).view(G, 1, 1)
                before = scale[b, :, j].view(G, 1, 1)
                if past:
                    two = torch.maximum(two, before)
                    codes[b, :, j, :past] = _nearest(codes[b, :, j, :past] * before / two)
                codes[b, :, j, past: past + t1 - t0] = _nearest(y / two)
                scale[b, :, j] = two.view(G)
        out[name] = codes.reshape(B, G, C, width) if name == "k" else codes.transpose(-1, -2).contiguous()
        out[name + "_scale"] = scale
    return out


def _exact_attend(s):
    """A sequence and a key / value head at a time, over the keys that it can see, some tokens at a time."""
    c = s["case"]
    B, S, H, G, D, V, C = c["B"], c["S"], c["H"], c["G"], c["D"], c["V"], c["C"]
    rep = H // G
    q, out = s["q"].view(B, S, G, rep, D), torch.zeros(B, S, G, rep, V, dtype=torch.float64, device="cuda")
    for b, (held, count) in enumerate(zip(s["held"].tolist(), s["counts"].tolist())):
        for g in range(G):
            k = (_values(s["k_codes"][b, g]).view(C // c["block"], -1) * s["k_scale"][b, g].double()[:, None]).view(C, D)
            v = (_values(s["v_codes"][b, g]) * s["v_scale"][b, g].double()[:, None, None]).transpose(1, 2).reshape(C, V)
            for t in range(0, count, 256):
                m = min(256, count - t)
                lo = max(0, held + t - c["window"] + 1) if c["window"] else 0
                hi = held + t + m
                j, p = torch.arange(lo, hi, device="cuda"), torch.arange(held + t, hi, device="cuda")[:, None]
                seen = (j <= p) & ((j > p - c["window"]) if c["window"] else (j >= 0))
                w = q[b, t:t + m, g].double().reshape(m * rep, D) @ k[lo:hi].T / math.sqrt(D)
                w = torch.softmax(w.view(m, rep, -1).masked_fill(~seen[:, None], -math.inf), -1)
                out[b, t:t + m, g] = (w.view(m * rep, -1) @ v[lo:hi]).view(m, rep, V)
    return out.view(B * S, H * V)
