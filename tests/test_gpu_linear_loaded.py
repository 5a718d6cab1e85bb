"""xb_linear_attention by chunks beside a memory system that is busy: what a chunk reads has arrived, however long its copies take."""
import numpy as np
import pytest
import torch

import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(128, 128), (128, 64), (64, 128), (64, 64)])
def test_beside_large_copies(dtype, dk, dv):
    """Lists of more than 20 chunks, a hundred calls while another stream copies gigabytes: the bits of a call on an idle GPU."""
    pkg.load()
    from x_deeplearning_b200 import ops
    rng = np.random.default_rng(dk)
    t = lambda *s: torch.from_numpy(rng.normal(0, 1, s).astype(np.float32)).to("cuda", T_[dtype])
    n, T, H = 24, 1500, 4
    q, k, v = t(n * T, H, dk), t(n * T, H, dk), t(n * T, H, dv)
    decay = torch.from_numpy(np.log1p(-np.exp2(-4.0 - np.arange(H))).astype(np.float32)).cuda()
    off = torch.arange(n + 1, device="cuda", dtype=torch.int32) * T
    a, b = torch.zeros(1 << 30, device="cuda", dtype=torch.uint8), torch.empty(1 << 30, device="cuda", dtype=torch.uint8)
    kw = dict(scale=dk ** -0.5, offsets=off, longest=T)
    want = ops.linear_attention(q, k, v, decay, **kw)
    torch.cuda.synchronize()
    beside = torch.cuda.Stream()
    with torch.cuda.stream(beside):
        for _ in range(60):
            b.copy_(a)
    outs = [torch.empty_like(want) for _ in range(4)]
    wrong = torch.zeros((), device="cuda", dtype=torch.int64)
    for i in range(100):
        y = ops.linear_attention(q, k, v, decay, out=outs[i % 4], **kw)
        wrong += (y != want).any()
    torch.cuda.synchronize()
    assert int(wrong) == 0
