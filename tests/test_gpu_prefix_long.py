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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 104])
@pytest.mark.parametrize("rows,rising", [(1, False), (1, True), (200, True)])
def test_long_sums(dtype, d, rows, rising):
    """4 000 000 keys of every head in pieces of one block, values about 3, with scores of one size or such that the maximum grows all the way. A weight is
    off by half a step, a result by one, and a sum by 2^-23 for each 16 of the 16 384 keys that the tensor cores add up at most; 2^-16 is left for the rest (exponentials 2^-21, scores
    2^-20, sums in fp32)."""
    pkg.load()
    from x_deeplearning_b200 import ops
    n, H = 1 << 22, 160
    n = n // 8 if rows > 1 else n
    g = torch.Generator(device="cuda").manual_seed(d)
    normal = lambda *s: torch.empty(s, device="cuda").normal_(generator=g)
    k, v = normal(n + H, d), normal(n + H, d) + 3
    if rising:
        k[:, 0] = torch.linspace(-40, 40, n + H, device="cuda")
    k, v = (t.to(dtype).flatten().as_strided((n, H, d), (d, d, 1)) for t in (k, v))
    q = normal(rows, H, d).to(dtype)
    q[:, :, 0] = 1.0
    y = ops.prefix_attention(q, T=1, prefix_k=k, prefix_v=v, scale=0.125)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    half = torch.finfo(dtype).eps / 2
    for h in (0, 77, 159):
        kh, vh = k[:, h].double(), v[:, h].double()
        for r in {0, rows // 2, rows - 1}:
            w = torch.softmax(kh @ q[r, h].double() * 0.125, 0)
            want, size = w @ vh, w @ vh.abs()
            assert ((y[r, h].double() - want).abs() <= size * (2 * half + 16_384 / 16 * 2.0 ** -23 + 2.0 ** -16)).all()
