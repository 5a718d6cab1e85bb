"""xb_prefix_attention on lists so long that a block's share of them takes seconds: its waits are for as long as work goes on."""
import pytest
import torch

import pkg

pytestmark = pytest.mark.gpu


def test_pieces_of_seconds():
    """160 heads of 8 that lie over one another in memory, 128 rows of a list with one own row beside 128 of one with 400 000 000: one of the two groups of warps
    waits while the other goes through these. One row in their middle has a score of 512 where the others have -512: it takes all."""
    pkg.load()
    from x_deeplearning_b200 import ops
    n, H, d = 3 << 27, 160, 8
    kv = torch.full(((n + H) * d,), -1.0, device="cuda", dtype=torch.float16)
    kv[n // 2 * d:(n // 2 + 1) * d] = 1.0
    kv = kv.as_strided((n, H, d), (d, d, 1))
    q = torch.full((256, H, d), 64.0, device="cuda", dtype=torch.float16)
    y = ops.prefix_attention(q, kv, kv, offsets=torch.tensor([0, 128, 256], dtype=torch.int32, device="cuda"),
                             own_offsets=torch.tensor([0, 1, n], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    assert (y[:127] == 0).all() and (y[127] == -1).all() and (y[128:] == 1).all()
