"""xb_prefix_attention where the two tiles of an item see different stretches of keys: each group of warps passes over what the other goes through, at its own
pace. Results against 64 bits, and the same bits in every run."""
import numpy as np
import pytest
import torch

import heads_oracle
from test_gpu_prefix import Call, _np, _pairs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("seed,H,Hkv,d", [(1, 15, 3, 96), (5, 15, 3, 96), (2, 12, 3, 80), (5, 12, 3, 80), (2, 2, 1, 128), (3, 2, 1, 128), (0, 1, 1, 72), (4, 1, 1, 72),
                                          (0, 8, 2, 64), (2, 8, 2, 64), (0, 5, 1, 40), (1, 5, 1, 40)])
def test_lists_with_rows_between(dtype, seed, H, Hkv, d):
    """Lists of a few queries with up to 1500 own rows, some of them long, some without queries, on a few prefixes."""
    rng = np.random.default_rng(seed)
    n = 130
    queries = np.floor(rng.exponential(14, n) * (rng.random(n) < 0.8)).astype(int)
    own = queries + np.where(rng.random(n) < 0.5, rng.integers(0, 300, n), 0) + np.where(rng.random(n) < 0.1, 1200, 0)
    c = Call(list(queries), list(own), [3, 500, 81, 0, 200], [20, 5, 30, 11, 29], H, Hkv, d, dtype, ahead=17, std=0.7, seed=seed)
    y = c.run()
    pick = [i for i in rng.permutation(n) if queries[i] > 0][:12]
    rows = np.concatenate([np.arange(c.off[i], c.off[i + 1]) for i in pick])
    at = np.r_[0, np.cumsum(queries[pick])]
    own_of, lists = _pairs(c.own_off), _pairs(at)
    want = heads_oracle.prefix(_np(c.q)[rows], _np(c.k), _np(c.v), lists, [own_of[i] for i in pick], [c.prefix_of[i] for i in pick], _np(c.pk), _np(c.pv), c.scale, dtype)
    heads_oracle.close(_np(y)[rows], *want, "y")
    for _ in range(20):
        assert torch.allclose(c.run().float(), y.float(), rtol=0.02, atol=0.02)
