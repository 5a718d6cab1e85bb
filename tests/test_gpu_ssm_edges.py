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


@pytest.mark.parametrize("value", ["nan", "inf"])
def test_a_broken_list_stays_broken(value):
    """A NaN (or an infinity) in the state stays to the list's end, whole or in chunks whose decay is nothing in fp32."""
    ops, capi = _ops()
    s, off, h = _two(np.random.default_rng(33))
    s["A"].fill_(-16.0)
    s["delta"].fill_(0.0)
    s["bias"].fill_(float(np.log(np.expm1(0.2))))               # steps of 0.2: a chunk of 64 rows decays by exp(-204)
    for longest in (5000, 0):
        assert _chunks(capi, 10000, 2, 40, 16, longest, capi.XB_F32)
        s["x"][100, :] = 1.0
        y, kept = _call(ops, s, off, h, longest, delta_bias=s["bias"])
        s["x"][100, :] = float(value)
        again, kept2 = _call(ops, s, off, h, longest, delta_bias=s["bias"])
        assert torch.equal(again[:100], y[:100]) and torch.equal(again[5000:], y[5000:]) and torch.equal(kept2[1], kept[1])
        assert not torch.isfinite(again[100:5000]).any() and not torch.isfinite(kept2[0]).any()
        # the same list alone, in rows enough lists that nothing is split
    n, t = 2000, 300
    rng = np.random.default_rng(34)
    w = _scan_inputs(rng, n * t, 0, 8, 4, 1, "f32", 0, 0)
    w["A"].fill_(-16.0)
    w["delta"].fill_(0.0)
    w["bias"].fill_(float(np.log(np.expm1(0.2))))
    w["x"][100] = float(value)
    y = ops.ssm_scan(w["x"], w["delta"], w["A"], w["B"], w["C"], delta_bias=w["bias"], T=t)
    assert not torch.isfinite(y[100:t]).any() and torch.isfinite(y[:100]).all() and torch.isfinite(y[t:]).all()


@pytest.mark.parametrize("A,h0", [(8.0, 0.0), (8.0, 1e-32), (-8.0, 1e30), (-8.0, 1.0)])
def test_chunks_whose_decay_fp32_does_not_hold(A, h0):
    """exp of a chunk's steps above 2^128 or below 2^-126 with a state that makes the product an ordinary number, or zero."""
    ops, capi = _ops()
    D, N, t = 8, 4, 6000
    rng = np.random.default_rng(35)
    s = _scan_inputs(rng, t, 0, D, N, 1, "f32", 0, 0)
    off = torch.tensor([0, t], dtype=torch.int32, device="cuda")
    assert _chunks(capi, t, 1, D, N, t, capi.XB_F32)
    s["A"].fill_(A)
    s["x"].zero_()
    s["delta"].zero_()
    s["delta"][960:1024] = 0.25                                 # 64 rows: exp(+-128) = 2^+-185
    h = torch.full((1, D, N), h0, device="cuda")
    y, kept = _call(ops, s, off, h, t, softplus=False)
    want, bound, last, elast = _scan_want(s, [(0, t)], 1, _np(h), "f32", bias=False, softplus=False)
    ssm_oracle.close(_np(y), want, bound, "y")
    ssm_oracle.close(_np(kept), np.stack(last), np.stack(elast), "states")
    assert h0 != 0 or (y == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("K", [2, 4])
@pytest.mark.parametrize("D,T", [(24, 1), (24, 40), (21, 40), (21, 1)])
def test_silu_of_sums_far_below_zero(dtype, K, D, T):
    """v sigmoid(v) goes to zero, whatever v: masks of the type's lowest value come out as zeros. Each beside ordinary values and NaN."""
    ops, capi = _ops()
    lowest = float(torch.finfo(T_[dtype]).min)
    far = [v for v in (-20.0, -41.0, -42.0, -50.0, -60.0, -80.0, -100.0, -1e4, -1e18, -1e30, lowest, lowest / 2, 41.0, 60.0, 100.0, 1e4, -lowest) if abs(v) <= -lowest]
    x = torch.randn(40, D, device="cuda", dtype=torch.float32)
    for i, v in enumerate(far):
        x[2 * i, (3 * i) % D] = v
        x[2 * i, (3 * i + 1) % D] = v
    x = x.to(T_[dtype])
    w = torch.zeros(D, K, device="cuda", dtype=T_[dtype])
    w[:, K - 1] = 1.0                                           # (the sums are the inputs)
    v = _np(x)
    with np.errstate(over="ignore"):
        want = v / (1 + np.exp(-v))
    # The sum is exact; exponential, quotient and products as ssm_oracle takes them, relative to the result (not to v). The exponential's
    # argument v log2(e) is off by the constant's rounding and the product's, 2^-24 relative each, so exp(v) by 2 |v| 2^-24 relative, which the
    # result shows where v < 0. Below -87 the quotient is flushed (1 + exp(-v) above 2^126): less than 2^-126 times |v| < 2^7 up to where
    # v exp(v) is itself below 2^-118.
    far_arg = np.where(v < 0, 2 * np.minimum(np.abs(v), 128) * 2.0 ** -24, 0)
    bound = (2.0 ** -20 + far_arg + ssm_oracle.HALF[dtype]) * np.abs(want) * (1 + 1e-3) + ssm_oracle.TINY[dtype] + 2.0 ** -118
    ssm_oracle.close(_np(ops.ssm_conv(x, w, T=T)), want, bound, dtype)
    x[7, 5] = float("nan")                                      # (its neighbours keep theirs)
    y = ops.ssm_conv(x, w, T=T)
    nan = y.isnan()
    assert nan[7, 5] and not nan[:, [c for c in range(D) if c != 5]].any()


def test_results_beside_their_inputs_and_over_them():
    """Columns of one matrix may hold both, the rows behind the last one too; the input itself may not."""
    ops, capi = _ops()
    rng = np.random.default_rng(37)
    for dtype in (torch.float32, torch.float16):
        m = torch.from_numpy(rng.normal(0, 1, (90, 48)).astype(np.float32)).cuda().to(dtype)
        w = torch.from_numpy(rng.normal(0, 1, (24, 4)).astype(np.float32)).cuda().to(dtype)
        for x, out in ((m[:90, :24], m[:90, 24:]), (m[:40, 24:], m[40:80, 24:]), (m[1:41, 24:], m[:40, :24]), (m[:1, 10:34], m[1:2, 10:34])):
            want = ops.ssm_conv(x.clone(), w)
            assert torch.equal(ops.ssm_conv(x, w, out=out), want)
        x = m[:40, :24]
        for out in (x, m[1:41, :24], m[:40, 1:25], m[:40, 23:47]):
            with pytest.raises(capi.XbError, match="overlaps"):
                ops.ssm_conv(x, w, out=out)
        A, B = -torch.rand(24, 16, device="cuda"), m[:40, 24:40].clone()
        with pytest.raises(capi.XbError, match="overlaps"):
            ops.ssm_scan(x, x.clone(), A, B, B, out=x)
        X, W = m[:40, :24], torch.zeros(24, 24, device="cuda", dtype=dtype)
        a = torch.zeros(2, 4, 24, device="cuda", dtype=dtype)
        ad = torch.zeros(40, device="cuda", dtype=torch.int32)
        with pytest.raises(capi.XbError, match="overlaps"):
            ops.lora_gemm(X, W, a, a.transpose(1, 2).contiguous(), ad, Y=X)
    st = torch.zeros(9, 3, 24, device="cuda")
    x, w = torch.zeros(8, 24, device="cuda"), torch.zeros(24, 4, device="cuda")
    with pytest.raises(capi.XbError, match="states overlap"):
        ops.ssm_conv(x, w, T=1, state_in=st[:8], state_out=st[1:])


def test_lists_behind_a_broken_one_keep_their_bits_in_the_convolution():
    ops, capi = _ops()
    rng = np.random.default_rng(36)
    off = torch.tensor([0, 5, 75, 75, 84, 384], dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b = (torch.from_numpy(rng.normal(0, 1, n).astype(np.float32)).cuda().to(dtype) for n in ((384, 40), (40, 4), (40,)))
        y = ops.ssm_conv(x, w, b, offsets=off)
        x[10:12] = float("inf")
        again = ops.ssm_conv(x, w, b, offsets=off)
        others = [r for r in range(384) if not 10 <= r < 15]
        assert torch.equal(again[others], y[others]) and not torch.isfinite(again[10:12]).all()


def test_scratch_that_the_device_does_not_have():
    """The allocator's error comes as torch's own calls raise it, and nothing is left behind. (The size is made up on the host.)"""
    ops, capi = _ops()
    m = capi.tensors()
    more = C.CFUNCTYPE(C.c_size_t, C.c_void_p)(lambda a: 1 << 50)
    m.bind("xb_ssm_scan_workspace_bytes", C.cast(more, C.c_void_p).value)
    x, A = torch.zeros(4, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    try:
        with pytest.raises(torch.OutOfMemoryError):
            ops.ssm_scan(x, x, A, x[:, :4], x[:, 4:])
    finally:
        m.bind("xb_ssm_scan_workspace_bytes", C.cast(capi.lib().xb_ssm_scan_workspace_bytes, C.c_void_p).value)
    assert (ops.ssm_scan(x, x, A, x[:, :4], x[:, 4:]) == 0).all()
