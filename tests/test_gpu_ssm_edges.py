"""xb_ssm_conv and xb_ssm_scan at the ends of their ranges: lists in many chunks beside broken ones, chunks whose decay fp32 does not hold,
sums far below zero. Against the formulas in 64 bits (tests/ssm_oracle.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

import pkg
import ssm_oracle
from test_gpu_ssm import T_, _np, _ops, _scan_inputs, _scan_want

pytestmark = pytest.mark.gpu


def _chunks(capi, rows, lists, D, N, longest, dtype):
    """Whether a call of these sizes walks its lists in chunks: only then it has scratch of this size"""
    a = capi.SsmScanArgs()
    a.x = a.delta = a.B = a.C = a.y = a.A = a.offsets = 4096
    a.rows, a.batch, a.D, a.N, a.groups, a.dtype, a.longest = rows, lists, D, N, 1, dtype, longest
    a.ldx = a.lddelta = a.ldy = D
    a.ldb = a.ldc = N
    return capi.lib().xb_ssm_scan_workspace_bytes(C.byref(a)) > 40 * D * N * 4


def _two(rng, D=40, N=16, t=5000):
    s = _scan_inputs(rng, 2 * t, 0, D, N, 1, "f32", 0, 0)
    off = torch.tensor([0, t, 2 * t], dtype=torch.int32, device="cuda")
    h = torch.from_numpy(rng.normal(0, 0.5, (2, D, N)).astype(np.float32)).cuda()
    return s, off, h


def _call(ops, s, off, h, longest, **k):
    kept = torch.full_like(h, 7.0)
    y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], offsets=off, longest=longest, h_in=h, h_out=kept, **k)
    return y, kept


@pytest.mark.parametrize("row", [10, 3000, 4700, 4900, 4980, 4999])
@pytest.mark.parametrize("what", ["delta", "x", "inf"])
def test_a_broken_list_and_the_next_in_many_chunks(row, what):
    """More chunks than the carry has parts, a border of lists inside one: the list behind a broken one keeps its bits."""
    ops, capi = _ops()
    s, off, h = _two(np.random.default_rng(31))
    assert _chunks(capi, 10000, 2, 40, 16, 5000, capi.XB_F32)
    y, kept = _call(ops, s, off, h, 5000, delta_bias=s["bias"])
    s["x" if what == "x" else "delta"][row] = float("inf" if what == "inf" else "nan")
    again, kept2 = _call(ops, s, off, h, 5000, delta_bias=s["bias"])
    assert torch.equal(again[5000:], y[5000:]) and torch.equal(kept2[1], kept[1])
    assert torch.equal(again[:row], y[:row]) and not torch.isfinite(again[row]).any()
    assert torch.isfinite(kept2[1]).all()


def test_growth_of_a_broken_list_and_the_next():
    """Steps given as they are, a list whose decay over a chunk overflows in fp32 ahead of an ordinary one."""
    ops, capi = _ops()
    s, off, h = _two(np.random.default_rng(32))
    s["A"].abs_().clamp_(min=1.0)
    s["delta"].uniform_(0, 0.002)
    y, kept = _call(ops, s, off, h, 5000, softplus=False)
    assert torch.isfinite(y[5000:]).all()
    s["delta"][4500:5000] = 4.0
    again, kept2 = _call(ops, s, off, h, 5000, softplus=False)
    assert torch.equal(again[5000:], y[5000:]) and torch.equal(kept2[1], kept[1])
