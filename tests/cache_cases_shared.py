"""An 8-bit cache on tensors that two holders go on from: each has what it appended, and neither sees the other's."""
import numpy as np

import cache_reference as R


def run_two_holders(be):
    rng = np.random.default_rng(3)
    G, D, V, block, capacity = 2, 64, 32, 16, 48
    x = [(rng.standard_normal((1, n, G * D)).astype(np.float32), rng.standard_normal((1, n, G * V)).astype(np.float32)) for n in (20, 5, 7)]
    hand = lambda i: (be.from_numpy(x[i][0]), be.from_numpy(x[i][1]))
    first = be.block_cache_append(*hand(0), be.empty_cache(1, G, D, V, capacity, block), position=0)
    second = be.block_cache_append(*hand(1), first, position=20)                                              # first is borrowed
    views = {n: be.reshape(t, t.shape) for n, t in second.items()}                                            # other handles of second's memory
    third = be.block_cache_append(*hand(2), {n: t.move() for n, t in second.items()}, position=25)
    again = be.block_cache_append(*hand(2), {n: t.move() for n, t in first.items()}, position=20)             # first's only holder gives it up
    for cache, appends in ((views, ((0, 0), (1, 20))), (third, ((0, 0), (1, 20), (2, 25))), (again, ((0, 0), (2, 20)))):
        k = (R.decode(be.to_vec(cache["k_codes"])).reshape(G, capacity, D) * np.repeat(be.to_vec(cache["k_scale"]).astype(np.float64), block).reshape(G, capacity, 1))
        v = R.decode(be.to_vec(cache["v_codes"])).reshape(G, capacity // block, V, block) * be.to_vec(cache["v_scale"]).astype(np.float64).reshape(G, -1, 1, 1)
        v = v.swapaxes(-1, -2).reshape(G, capacity, V)
        for g in range(G):
            heads = R.Head(capacity, D, block), R.Head(capacity, V, block)
            for i, at in appends:
                heads[0].append(at, x[i][0][0, :, g * D: (g + 1) * D])
                heads[1].append(at, x[i][1][0, :, g * V: (g + 1) * V])
                end = at + x[i][0].shape[1]
            np.testing.assert_array_equal(k[g, :end], heads[0].x[:end])
            np.testing.assert_array_equal(v[g, :end], heads[1].x[:end])
