"""xb_prefix_attention where a block's pieces of work are a tile alone and then two, of which one sees no keys: the group of warps that has nothing to do
waits for its turn. Results against 64 bits, many runs."""
import numpy as np
import pytest
import torch

import heads_oracle
from test_gpu_prefix import Call, _np, _pairs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,d", [(1, 1, 40), (2, 1, 64), (12, 3, 64), (8, 2, 48), (1, 1, 72), (2, 1, 128), (12, 3, 80), (8, 2, 104)])
@pytest.mark.parametrize("seed", range(5))
def test_pieces_of_few_blocks(dtype, H, Hkv, d, seed):
    rng = np.random.default_rng(seed)
    n = 130
    queries = np.floor(rng.exponential(14, n) * (rng.random(n) < 0.8)).astype(int)
    own = queries + np.where(rng.random(n) < 0.5, rng.integers(0, 300, n), 0) + np.where(rng.random(n) < 0.1, 1200, 0)
    c = Call(list(queries), list(own), [3, 500, 81, 0, 200], [20, 5, 30, 11, 29], H, Hkv, d, dtype, ahead=17, std=0.7, seed=seed)
    y = c.run()
    pick = [i for i in rng.permutation(n) if queries[i] > 0][:12]
    rows = np.concatenate([np.arange(c.off[i], c.off[i + 1]) for i in pick])
    own_of = _pairs(c.own_off)
    want = heads_oracle.prefix(_np(c.q)[rows], _np(c.k), _np(c.v), _pairs(np.r_[0, np.cumsum(queries[pick])]), [own_of[i] for i in pick], [c.prefix_of[i] for i in pick],
                               _np(c.pk), _np(c.pv), c.scale, dtype)
    heads_oracle.close(_np(y)[rows], *want, "y")
    for _ in range(30):
        assert torch.equal(c.run(), y)
