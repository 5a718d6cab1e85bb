"""xb_linear_attention on values of very different sizes side by side: columns of values and states, rows of queries, states near fp32's end. What
a value is off by goes by the sums that it is part of, not by its neighbours (bounds from tests/heads_oracle.py, element by element)."""
import numpy as np
import pytest
import torch

import heads_oracle
import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16}
SIZES = [(64, 64), (128, 128), (40, 72)]
LISTS = [(0, 200), (200, 270), (270, 1570)]


def _ops():
    pkg.load()
    from x_deeplearning_b200 import ops
    return ops


def _np(t):
    return t.detach().double().cpu().numpy()


def _check(q, k, v, h, scale, dtype, slowest=4.0):
    ops = _ops()
    H, n = q.shape[1], len(LISTS)
    ld = torch.from_numpy(np.log1p(-np.exp2(-slowest - 5 * np.arange(H))).astype(np.float32)).cuda()
    off = torch.tensor([0] + [e for _, e in LISTS], dtype=torch.int32, device="cuda")
    kept = torch.empty(n, H, q.shape[2], v.shape[2], device="cuda")
    y = ops.linear_attention(q, k, v, ld, scale=scale, offsets=off, h_in=h, h_out=kept)
    h0 = np.zeros(kept.shape) if h is None else _np(h)
    want, bound, last, elast = heads_oracle.linear(_np(q), _np(k), _np(v), _np(ld), scale, LISTS, h0, dtype)
    # (what the type holds: where the bound goes past its end, 65504 in fp16, a right result may be infinite)
    ok = np.abs(want) + bound < (60000 if dtype == "f16" else 1e38)
    assert ok.mean() > 0.3
    heads_oracle.close(_np(y)[ok], want[ok], bound[ok], "y")
    heads_oracle.close(_np(kept), np.stack(last), np.stack(elast), "states")


def _sizes(n, lo, hi, seed):
    """Powers of two from 2^lo to 2^hi in any order"""
    return torch.from_numpy(np.exp2(np.random.default_rng(seed).permutation(np.round(np.linspace(lo, hi, n))))).float().cuda()


def _normal(*shape, seed):
    return torch.from_numpy(np.random.default_rng(seed).normal(0, 1, shape)).float().cuda()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dk,dv", SIZES)
def test_columns_of_values(dtype, dk, dv):
    q, k, v = _normal(1570, 2, dk, seed=1), _normal(1570, 1, dk, seed=2), _normal(1570, 1, dv, seed=3)
    v = v.clamp(-3.5, 3.5) * _sizes(dv, -13, 14, 4)
    _check(*(t.to(T_[dtype]) for t in (q, k, v)), None, 1.0, dtype)
    _check(*(t.to(T_[dtype]) for t in (q, k, v)), None, 2.0 ** -10, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dk,dv", SIZES)
def test_columns_of_kept_states(dtype, dk, dv):
    q, k, v = _normal(1570, 2, dk, seed=1), _normal(1570, 1, dk, seed=2), _normal(1570, 1, dv, seed=3)
    h = _normal(3, 2, dk, dv, seed=5) * _sizes(dv, -10, 40, 6)
    _check(*(t.to(T_[dtype]) for t in (q, k, v)), h, 1.0, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dk,dv", SIZES)
def test_rows_of_queries(dtype, dk, dv):
    q, k, v = _normal(1570, 2, dk, seed=1), _normal(1570, 1, dk, seed=2), _normal(1570, 1, dv, seed=3)
    q = q.clamp(-3.5, 3.5) * _sizes(1570, -13, 14, 7)[:, None, None]
    for big in (1.0, 2.0 ** 12):
        _check(*(t.to(T_[dtype]) for t in (q, k.clamp(-3.5, 3.5) * big, v)), None, 1.0 / big, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-26, 1e-20, 1e20, 1e30, 1e33, 1e36])
def test_states_near_the_end_of_fp32(dtype, size):
    q, k, v = _normal(1570, 2, 64, seed=1), _normal(1570, 1, 64, seed=2), _normal(1570, 1, 64, seed=3)
    h = (_normal(3, 2, 64, 64, seed=5).double() * size).float()
    if size < 1:
        k, v = k * 0, v * 0                                              # (else nothing of the kept states would be left to see)
    _check(*(t.to(T_[dtype]) for t in (q, k, v)), h, 1.0 / size, dtype, slowest=9.0)
