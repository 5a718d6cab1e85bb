"""xb_prefix_attention: a row's bits do not depend on what calls before it left in shared memory (heads that share keys in numbers that do not divide 128)."""
import numpy as np
import pytest
import torch

import pkg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("share,Hkv,d", [(5, 1, 40), (7, 2, 128), (33, 1, 64), (99, 1, 128), (3, 3, 112), (43, 1, 8)])
def test_same_bits_after_other_calls(dtype, share, Hkv, d):
    pkg.load()
    from x_deeplearning_b200 import ops
    rng = np.random.default_rng(share)
    t = lambda *s, std=1.0: torch.from_numpy(rng.normal(0, std, s)).to("cuda", dtype)
    rows, n = 300, 3000
    q, k, v, pk, pv = t(rows, share * Hkv, d), t(rows, Hkv, d), t(rows, Hkv, d), t(n, Hkv, d), t(n, Hkv, d)
    kw = dict(T=2, prefix_k=pk, prefix_v=pv, scale=2.0 * d ** -0.5)
    want = ops.prefix_attention(q, k, v, **kw)
    other = t(20_000, 1, 128, std=100.0)
    for i in range(12):
        # (results of every size, infinities among them, where this call's queries will lie)
        ops.prefix_attention(other, other, other * (10.0 ** (i - 6)) if i < 11 else other * float("inf"), T=1)
        assert torch.equal(ops.prefix_attention(q, k, v, **kw), want)
    assert ops.device_status() == 0
