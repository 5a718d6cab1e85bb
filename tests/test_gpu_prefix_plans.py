"""xb_prefix_attention on offsets and members that do not ascend or point outside: what the device finds there changes results, never memory beside them."""
import numpy as np
import pytest
import torch

import pkg

pytestmark = pytest.mark.gpu


def _ops():
    pkg.load()
    from x_deeplearning_b200 import ops
    return ops


def _cuda(a):
    return torch.from_numpy(np.asarray(a, np.int32)).cuda()


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 64), (3, 1, 128)])
def test_what_does_not_ascend(seed, H, Hkv, d):
    ops = _ops()
    rng = np.random.default_rng(seed)
    t = lambda *s: torch.from_numpy(rng.normal(size=s)).to("cuda", torch.bfloat16)
    batch, prefixes, rows, own, prefix = (int(n) for n in (rng.integers(1, 60), rng.integers(1, 7), rng.integers(1, 900), rng.integers(1, 2500), rng.integers(1, 3000)))
    q, k, v, pk, pv = t(rows, H, d), t(own, Hkv, d), t(own, Hkv, d), t(prefix, Hkv, d), t(prefix, Hkv, d)

    def wild(n, most):
        a = rng.integers(0, most + 1, n)
        a[rng.random(n) < 0.1] = rng.choice([-5, -2**31, 2**31 - 1])
        return a
    around = torch.full((rows + 512, H, d), 5.0, device="cuda", dtype=torch.bfloat16)
    args = dict(offsets=_cuda(wild(batch + 1, rows)), own_offsets=_cuda(wild(batch + 1, own)), members=_cuda(wild(prefixes + 1, batch)),
                prefix_offsets=_cuda(wild(prefixes + 1, prefix)), prefix_k=pk, prefix_v=pv, scale=d ** -0.5)
    for names in ((), ("members",), ("offsets",), ("offsets", "own_offsets"), ("members", "prefix_offsets")):
        # (those named in ascending order, the others as they are)
        kw = {n: torch.sort(a)[0] if n in names else a for n, a in args.items()}
        ops.prefix_attention(q, k, v, out=around[256:256 + rows], **kw)
        torch.cuda.synchronize()
        assert ops.device_status() == 0
        assert (around[:256] == 5.0).all() and (around[256 + rows:] == 5.0).all()
        assert not torch.isnan(around.float()).any()          # (every key and value that there is is finite)
