"""xb_prefix_attention beside a memory system that is busy: whatever is late, the bits are those of a call on an idle GPU."""
import numpy as np
import pytest
import torch

import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lists,own,prefix", [(512, 1, 20_000), (60, 100, 400)])
def test_beside_large_copies(dtype, d, lists, own, prefix):
    pkg.load()
    from x_deeplearning_b200 import ops
    rng = np.random.default_rng(d)
    t = lambda *s: torch.from_numpy(rng.normal(0, 1, s).astype(np.float32)).to("cuda", T_[dtype])
    rows = lists * own
    q, k, v, pk, pv = t(rows, 4, d), t(rows, 2, d), t(rows, 2, d), t(prefix, 2, d), t(prefix, 2, d)
    a, b = torch.zeros(1 << 30, device="cuda", dtype=torch.uint8), torch.empty(1 << 30, device="cuda", dtype=torch.uint8)
    kw = dict(T=own, prefix_k=pk, prefix_v=pv, scale=d ** -0.5)
    want = ops.prefix_attention(q, k, v, **kw)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(60):
            b.copy_(a)
    outs = [torch.empty_like(want) for _ in range(4)]
    wrong = torch.zeros((), device="cuda", dtype=torch.int64)
    for i in range(100):
        wrong += (ops.prefix_attention(q, k, v, out=outs[i % 4], **kw) != want).any()
    torch.cuda.synchronize()
    assert int(wrong) == 0 and ops.device_status() == 0
