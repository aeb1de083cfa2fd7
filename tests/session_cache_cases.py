"""Dense checkpoints whose keys and values are held as 8-bit codes: what a session answers, held to the model's mathematics in 64-bit numpy
over the same cache.  Codes are rounded, so an error of a key too small to see elsewhere may move a code by a whole step: results may differ
by what the model itself moves by when its keys and values are off by rounding errors (`allowed`)."""
import numpy as np

import cache_reference as R
from model_cases import TINY_LLAMA, TINY_QWEN3, params_of
from np_models import _Wide, rmsnorm

SCALING = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 32},
    "yarn": {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32},
}
MODELS = {"llama": TINY_LLAMA, "qwen3": TINY_QWEN3}


def config(cfg, scaling="none", **more):
    c = {"model_type": cfg.arch, "hidden_size": cfg.hidden_size, "num_hidden_layers": cfg.num_hidden_layers, "num_attention_heads": cfg.num_attention_heads,
         "num_key_value_heads": cfg.num_key_value_heads, "intermediate_size": cfg.intermediate_size, "vocab_size": cfg.vocab_size, "head_dim": cfg.hd,
         "rms_norm_eps": cfg.rms_norm_eps, "rope_theta": cfg.rope_theta, "tie_word_embeddings": cfg.tie_word_embeddings, "kv_cache": "f8", **more}
    if SCALING[scaling]:
        c["rope_scaling"] = SCALING[scaling]
    return c


def load(session, cfg, params, scaling="none", **more):
    session.clear_params()
    session.load_config(config(cfg, scaling, **more))
    for name, w in params.items():
        session.set_param(name, w)


def turns(cfg, scaling):
    """Frequencies (turns a position) and magnitude of a head's pairs, from the published formulas of the three scalings."""
    d, base, s = cfg.hd, cfg.rope_theta, SCALING[scaling]
    f = base ** -(np.arange(0, d, 2) / d) / (2 * np.pi)
    if not s:
        return f, 1.0
    kind, factor = s.get("rope_type", s.get("type")), s["factor"]
    if kind == "linear":
        return f / factor, 1.0
    times = f * s["original_max_position_embeddings"]  # of a whole turn within the positions that the model has learnt
    if kind == "llama3":
        keep = np.clip((times - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"]), 0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    pair = lambda t: d * np.log(s["original_max_position_embeddings"] / (t * 2 * np.pi)) / (2 * np.log(base))
    low, high = max(np.floor(pair(32.0)), 0), min(np.ceil(pair(1.0)), d - 1)
    down = np.clip((np.arange(d // 2) - low) / max(high - low, 0.001), 0, 1)
    return f / factor * down + f * (1 - down), 0.1 * np.log(factor) + 1.0


class Reference:
    """The model with a cache, one sequence."""

    def __init__(self, cfg, params, scaling="none", noise=None):
        self.c, self.P, self.noise, self.held = cfg, _Wide(params), noise, 0
        self.turns, self.magnitude = turns(cfg, scaling)
        self.k, self.v = ([[R.Head(1024, cfg.hd, 64) for _ in range(cfg.num_key_value_heads)] for _ in range(cfg.num_hidden_layers)] for _ in range(2))

    def off(self, x):
        return x if self.noise is None else x * (1 + 2.0 ** -17 * self.noise.uniform(-1, 1, x.shape))

    def step(self, tokens):
        c, P, r = self.c, self.P, self.c.arch
        x, S, group = P[f"{r}.model.embed_tokens.weight"][tokens], len(tokens), c.num_attention_heads // c.num_key_value_heads
        pos = self.held + np.arange(S)
        for l in range(c.num_hidden_layers):
            p = f"{r}.model.layers.{l}"
            h = rmsnorm(x, P[f"{p}.input_layernorm.weight"], c.rms_norm_eps)
            q, k, v = ((h @ P[f"{p}.self_attn.{n}_proj.weight"].T).reshape(S, -1, c.hd) for n in "qkv")
            if r == "qwen3":
                q, k = (rmsnorm(y, P[f"{p}.self_attn.{n}_norm.weight"], c.rms_norm_eps) for n, y in (("q", q), ("k", k)))
            q, k = (R.rotate(y, pos, self.turns, self.magnitude, False) for y in (q, k))
            k, v = self.off(k), self.off(v)
            out = np.zeros((S, c.num_attention_heads, c.hd))
            for g in range(c.num_key_value_heads):
                self.k[l][g].append(self.held, k[:, g])
                self.v[l][g].append(self.held, v[:, g])
                for s in range(S):
                    heads = slice(g * group, (g + 1) * group)
                    out[s, heads] = R.attend(q[s, heads], pos[s], self.k[l][g].x, self.v[l][g].x, c.hd ** -0.5, 0)[0]
            x = x + out.reshape(S, -1) @ P[f"{p}.self_attn.o_proj.weight"].T
            h = rmsnorm(x, P[f"{p}.post_attention_layernorm.weight"], c.rms_norm_eps)
            gate = h @ P[f"{p}.mlp.gate_proj.weight"].T
            x = x + (gate / (1 + np.exp(-gate)) * (h @ P[f"{p}.mlp.up_proj.weight"].T)) @ P[f"{p}.mlp.down_proj.weight"].T
        self.held += S
        head = f"{r}.model.embed_tokens.weight" if c.tie_word_embeddings else f"{r}.lm_head.weight"
        return rmsnorm(x, P[f"{r}.model.norm.weight"], c.rms_norm_eps) @ P[head].T


def answers(cfg, params, steps, scaling="none"):
    """(logits of every step, how far a session's may be off)."""
    exact = Reference(cfg, params, scaling)
    logits = [exact.step(t) for t in steps]
    # The keys and values of a session are off by the roundings of 32-bit products over <= 160 terms and of the norms, at most
    # 200 * 2^-24 < 2^-16 of a typical term.  Three draws of errors within 2^-17 move about as many codes as those roundings do; any one
    # code counts alike, so a session may be off by four times the farthest of the three, beside the 1e-3 that the products of a model
    # may differ by from 64 bits anywhere (tests/test_oracle_models.py).
    moved = 0.0
    for seed in range(3):
        near = Reference(cfg, params, scaling, np.random.default_rng(seed))
        moved = max(moved, max(np.abs(near.step(t) - e).max() for t, e in zip(steps, logits)))
    return logits, 4 * moved + 1e-3 * max(np.abs(e).max() for e in logits)


def tokens_of(cfg, lengths, seed):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, cfg.vocab_size, n).astype(np.uint32) for n in lengths]


def run_steps(session, name, lengths, scaling="none", max_positions=0):
    """A request in portions: every place's logits."""
    cfg = MODELS[name]
    params = params_of(cfg, seed=3, scale=4.0)
    load(session, cfg, params, scaling)
    steps = tokens_of(cfg, lengths, 7)
    want, allowed = answers(cfg, params, steps, scaling)
    for n, (t, w) in enumerate(zip(steps, want)):
        got = session.step(5, t, rows=range(len(t)), max_positions=max_positions)
        assert np.abs(got - w).max() <= allowed, (n, np.abs(got - w).max(), allowed)
    session.end(5)


def run_interleaved(session):
    """Requests of different lengths in turn answer what each answers alone, bit for bit."""
    cfg = MODELS["llama"]
    params = params_of(cfg, seed=3, scale=4.0)
    load(session, cfg, params)
    parts = {1: tokens_of(cfg, (3, 1, 60, 1), 1), 2: tokens_of(cfg, (65, 1, 1, 2), 2), 3: tokens_of(cfg, (1, 1, 1, 1), 3)}
    alone = {r: [session.step(r, t, rows=range(len(t))) for t in p] for r, p in parts.items()}
    for r in parts:
        session.end(r)
    for n in range(4):
        for r, p in parts.items():
            np.testing.assert_array_equal(session.step(r, p[n], rows=range(len(p[n]))), alone[r][n])
    for r in parts:
        session.end(r)


def run_generate(session, name):
    """Greedy choices of a batch are those of each sequence alone, and those of the reference where it is decided."""
    cfg = MODELS[name]
    params = params_of(cfg, seed=5, scale=4.0)
    load(session, cfg, params)
    prompt = np.stack(tokens_of(cfg, (61, 61), 4))
    toks, _ = session.generate(prompt, steps=8, max_positions=69)
    for b in range(2):
        steps = [prompt[b]] + [toks[n, b:b + 1] for n in range(8)]
        want, allowed = answers(cfg, params, steps)
        for n, w in enumerate(want):
            row = w[-1]
            assert row[toks[n, b]] >= row.max() - 2 * allowed, (b, n)


def run_schedules(session, same):
    """Recorded runs copy the cache where plain ones write into it; the answers are the same."""
    cfg = MODELS["qwen3"]
    params = params_of(cfg, seed=5, scale=4.0)
    load(session, cfg, params)
    steps, got = tokens_of(cfg, (7, 1, 70, 1), 9), []
    try:
        for schedule in range(3):
            session.set_schedule(schedule)
            got.append([session.step(1, t, rows=range(len(t))) for t in steps])
            session.end(1)
    finally:
        session.set_schedule(0)
    for g in got[1:]:
        for a, b in zip(g, got[0]):
            same(a, b)
