"""xb_qk_norm_rope against its formula in 64 bits (tests/heads_oracle.py, where the bounds come from)."""
import numpy as np
import pytest
import torch

import heads_oracle
import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    pkg.load()
    from x_deeplearning_b200 import capi, ops
    return ops, capi


def _np(t):
    return t.detach().double().cpu().numpy()


def _freqs(rot):
    return torch.exp(torch.arange(rot // 2, dtype=torch.float64) * (-np.log(10000.0) / max(rot // 2, 1))).float().cuda()


def _check(q, k, positions, freqs, wq=None, wk=None, eps=1e-6, norm=True, adjacent=False, dtype="f32", out=None):
    ops, _ = _ops()
    want = [heads_oracle.rope(_np(x), positions.cpu().numpy(), None if freqs is None else _np(freqs), None if w is None else _np(w), eps, norm, adjacent, dtype)
            for x, w in ((q, wq), (k, wk)) if x is not None]
    oq, ok = out or (None, None)
    got = ops.qk_norm_rope(q, k, positions, freqs, q_weight=wq, k_weight=wk, eps=eps, norm=norm, adjacent=adjacent, out_q=oq, out_k=ok)
    assert (got[1] is None) == (k is None)
    for name, g, (y, e) in zip("qk", got, want):
        heads_oracle.close(_np(g), y, e, name)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 3, 257])
@pytest.mark.parametrize("Hq,Hk,d,rot", [(1, 1, 2, 2), (8, 2, 64, 64), (3, 1, 36, 36), (5, 0, 72, 16), (4, 4, 128, 128), (2, 1, 256, 256), (3, 3, 50, 20),
                                         (1, 1, 255, 254), (33, 7, 16, 8), (2, 2, 40, 0)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_formula(dtype, rows, Hq, Hk, d, rot, adjacent):
    rng = np.random.default_rng(rows + d)
    t = lambda *s, std=1.5: torch.from_numpy(rng.normal(0, std, s)).to("cuda", T_[dtype])
    positions = torch.from_numpy(rng.integers(0, 1 << 20, rows).astype(np.int32)).cuda()
    wq, wk = torch.from_numpy(rng.normal(1, 0.2, (2, d)).astype(np.float32)).cuda()
    freqs = _freqs(rot)
    q, k = t(rows, Hq, d), t(rows, Hk, d) if Hk else None
    _check(q, k, positions, freqs, wq, wk if Hk else None, adjacent=adjacent, dtype=dtype)
    # slices of one projection; no weights, a large eps; and in place
    qkv = t(rows, Hq + 2 * Hk + 1, d)
    q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hk] if Hk else None
    _check(q, k, positions, freqs, eps=0.25, adjacent=adjacent, dtype=dtype)
    _check(q, k, positions, freqs, norm=False, adjacent=adjacent, dtype=dtype)
    rest = qkv[:, Hq + Hk:].clone()
    fresh = _check(q, k, positions, freqs, wq, wk if Hk else None, adjacent=adjacent, dtype=dtype)
    here = _check(q, k, positions, freqs, wq, wk if Hk else None, adjacent=adjacent, dtype=dtype, out=(q, k))
    assert torch.equal(here[0], fresh[0]) and (not Hk or torch.equal(here[1], fresh[1]))
    assert torch.equal(qkv[:, Hq + Hk:], rest)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_strides(dtype):
    """Rows and heads anywhere: heads outside rows, rows that start off 16 bytes, a row stride of 0 among the inputs, results into wider rows."""
    rng = np.random.default_rng(5)
    rows, H, d = 37, 3, 64
    base = torch.from_numpy(rng.normal(0, 1, (H, rows, d))).to("cuda", T_[dtype])
    positions = torch.arange(rows, device="cuda", dtype=torch.int32) - 5                # (negative positions too)
    freqs = _freqs(d)
    _check(base.transpose(0, 1), None, positions, freqs, dtype=dtype)
    wide = torch.from_numpy(rng.normal(0, 1, (rows, H * d + 3))).to("cuda", T_[dtype])
    off = wide[:, 1:1 + H * d].unflatten(1, (H, d))
    _check(off, None, positions, freqs, dtype=dtype)
    _check(base[:, :1].transpose(0, 1).expand(rows, H, d), None, positions, freqs, dtype=dtype)
    out = torch.full((rows, 2 * H + 1, d), 9.0, device="cuda", dtype=T_[dtype])
    _check(off, base.transpose(0, 1), positions, freqs, dtype=dtype, out=(out[:, :H], out[:, H + 1:]))
    assert (out[:, H] == 9.0).all()


def test_far_positions():
    """Angles of far positions are those of 64 bits: fp32 keeps 2^-24 of an angle of 2^24."""
    positions = torch.tensor([0, 1, 16777215, 16777217, 2000000011, -2000000011], device="cuda", dtype=torch.int32)
    q = torch.zeros(6, 1, 32, device="cuda")
    q[:, :, :16] = 1
    _check(q, None, positions, _freqs(32), norm=False)
    _check(q, None, positions, torch.full((16,), 1.0, device="cuda"), norm=False, adjacent=True)


def test_values_at_the_ends():
    """Zeros under a norm without eps are 0 / 0; a NaN stays in its head; no rows and no heads are calls that do nothing."""
    ops, _ = _ops()
    q = torch.ones(4, 2, 32, device="cuda", dtype=torch.float16)
    q[1, 0, 3] = float("nan")
    q[2, 1] = 0
    pos, f = torch.zeros(4, dtype=torch.int32, device="cuda"), _freqs(32)
    y, none = ops.qk_norm_rope(q, None, pos, f)
    assert none is None and torch.isnan(y[1, 0]).all() and not torch.isnan(y[1, 1]).any() and (y[2, 1] == 0).all() and (y[0] == 1).all()
    assert torch.isnan(ops.qk_norm_rope(q, None, pos, f, eps=0.0)[0][2, 1]).all()
    y, k = ops.qk_norm_rope(q[:0], q[:0], pos[:0], f)
    assert y.shape == (0, 2, 32) and k.shape == (0, 2, 32)
    # the norm alone
    y, _ = ops.qk_norm_rope(q, None, None, None)
    assert (y[0] == 1).all()


def test_captured_and_on_other_streams():
    ops, _ = _ops()
    rng = np.random.default_rng(2)
    q = torch.from_numpy(rng.normal(0, 1, (500, 4, 64)).astype(np.float32)).cuda().half()
    pos, f = torch.arange(500, device="cuda", dtype=torch.int32), _freqs(64)
    want, _ = ops.qk_norm_rope(q, None, pos, f)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.qk_norm_rope(q, None, pos, f, out_q=out)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.qk_norm_rope(q, None, pos, f, out_q=out)
    q.mul_(-1)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -want)
