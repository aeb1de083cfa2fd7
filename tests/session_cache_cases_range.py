"""A session over the 8-bit cache whose texts hold tokens without a value: their rows of the embedding are zero, as those of padding may be."""
import numpy as np

import session_cache_cases as cases
from model_cases import params_of


def run_tokens_of_zeros(session, name):
    cfg = cases.MODELS[name]
    params = params_of(cfg, seed=3, scale=4.0)
    table = params[f"{cfg.arch}.model.embed_tokens.weight"] = params[f"{cfg.arch}.model.embed_tokens.weight"].copy()
    table[0] = 0.0
    cases.load(session, cfg, params)
    text = 1 + cases.tokens_of(cfg, (64 + 40,), 7)[0] % (cfg.vocab_size - 1)
    # 64 tokens, two blocks of zeros at least for each of the waves that a step is taken by, and more tokens (fewer than 1024: the reference holds no more)
    steps = [np.concatenate([text[:64], np.zeros(576, np.uint32), text[64:102]]).astype(np.uint32), text[102:103], text[103:104]]
    want, allowed = cases.answers(cfg, params, steps)
    for n, (t, w) in enumerate(zip(steps, want)):
        rows = [r for r in (0, 63, 64, 200, 600, 639, 640, len(t) - 1) if r < len(t)]
        got = session.step(5, t, rows=rows)
        assert np.abs(got - w[rows]).max() <= allowed, (n, np.abs(got - w[rows]).max(), allowed)
    session.end(5)
