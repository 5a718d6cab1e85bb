"""Calls of ops.ssm_conv, ops.ssm_scan, ops.lora_gemm and their C functions that are refused before anything runs: scratch that is not
there, sizes that 32-bit counts do not hold, results over their own inputs. Host logic alone."""
import ctypes as C

import pytest
import torch

import pkg
from test_ssm_lora_binding import bound  # noqa: F401  (a fixture)


def test_scratch_whose_bytes_are_one(bound):  # noqa: F811
    """An expanded vector has many elements and one byte."""
    ops, capi, seen, need, _ = bound
    x, w = torch.zeros(12, 24, dtype=torch.float16), torch.zeros(1, dtype=torch.uint8).expand(4096)
    need[0] = 1000
    with pytest.raises(capi.XbError, match="workspace"):
        ops.ssm_scan(x, x, torch.zeros(24, 16), x[:, :16], x[:, :16], workspace=w)
    with pytest.raises(capi.XbError, match="workspace"):
        ops.lora_gemm(x, torch.zeros(16, 24, dtype=torch.float16), torch.zeros(3, 8, 24, dtype=torch.float16), torch.zeros(3, 16, 8, dtype=torch.float16),
                      torch.zeros(12, dtype=torch.int32), trans_b=True, workspace=w)
    assert not seen
    ops.ssm_scan(x, x, torch.zeros(24, 16), x[:, :16], x[:, :16], workspace=torch.zeros(4096, dtype=torch.uint8)[:1])
    assert seen[-1][1][1] == 1


AT, ARG, LIMIT = 4096, -1, -5


def _conv(c, **k):
    a = c.SsmConvArgs()
    a.x = a.y = a.w = AT
    a.y += 1 << 20
    a.rows, a.batch, a.D, a.K, a.dtype, a.ldx, a.ldy = 12, 3, 24, 4, c.XB_F16, 24, 24
    for n, v in k.items():
        setattr(a, n, v)
    return a


def _scan(c, **k):
    a = c.SsmScanArgs()
    a.x = a.delta = a.B = a.C = a.A = AT
    a.y = AT + (1 << 20)
    a.rows, a.batch, a.D, a.N, a.groups, a.dtype = 12, 3, 24, 16, 2, c.XB_BF16
    a.ldx = a.lddelta = a.ldy = 24
    a.ldb = a.ldc = 32
    for n, v in k.items():
        setattr(a, n, v)
    return a


def _lora(c, **k):
    a = c.LoraArgs()
    a.X = a.W = a.A = a.B = a.adapter = AT
    a.Y = AT + (1 << 20)
    a.M, a.N, a.K, a.r, a.n_adapters, a.trans_w, a.dtype, a.y_dtype = 10, 16, 32, 8, 3, 1, c.XB_F16, c.XB_F16
    a.ldx = a.ldw = a.lda = 32
    a.ldy, a.ldb, a.stride_a, a.stride_b = 16, 8, 256, 128
    for n, v in k.items():
        setattr(a, n, v)
    return a


def test_channels_and_lists_that_round_up_past_32_bits():
    m = pkg.load()
    c, L = m.capi, m.lib()
    most = (1 << 31) - 1
    for k in (dict(D=most, ldx=most, ldy=most), dict(D=most - 1022, ldx=most, ldy=most), dict(batch=most, rows=4, offsets=AT), dict(batch=most, rows=0)):
        assert L.xb_ssm_conv(C.byref(_conv(c, **k)), None) == LIMIT, k
        assert b"xb_ssm_conv" in L.xb_last_error()
    for k in (dict(D=most, groups=1, ldx=most, ldy=most, lddelta=most), dict(batch=most, rows=4, offsets=AT), dict(batch=most - 1022, rows=0)):
        a = _scan(c, **k)
        assert L.xb_ssm_scan_workspace_bytes(C.byref(a)) == 0 and L.xb_ssm_scan(C.byref(a), None, 0, None) == LIMIT, k
        assert b"xb_ssm_scan" in L.xb_last_error()


def test_adapters_whose_scratch_passes_64_bits():
    """Adapters that share their memory (strides of 0 and 1) are a small tensor; what is laid out of them is not."""
    m = pkg.load()
    c, L = m.capi, m.lib()
    most = (1 << 31) - 1024
    for k in (dict(M=most, N=most, ldy=most, n_adapters=most, r=128, ldb=128, stride_a=0, stride_b=1),
              dict(M=most, K=most, ldx=most, ldw=most, lda=most, n_adapters=most, r=128, ldb=128, stride_a=1, stride_b=0)):
        a = _lora(c, **k)
        assert L.xb_lora_workspace_bytes(C.byref(a)) == 0, k
        assert L.xb_lora_gemm(C.byref(a), AT, 1 << 60, None) == LIMIT, k
        assert b"xb_lora_gemm" in L.xb_last_error()


def test_results_over_inputs():
    m = pkg.load()
    c, L = m.capi, m.lib()
    row = 24 * 2
    for k in (dict(y=AT), dict(y=AT + 2), dict(y=AT + 5 * row), dict(y=AT + 11 * row + 46), dict(x=AT + row), dict(y=AT, ldy=40), dict(ldx=100, ldy=100, y=AT + 46),
              dict(ldx=40, ldy=40, y=AT + 34), dict(ldx=40, ldy=40, y=AT + 3 * 80 + 34)):
        k = {**dict(y=AT), **k} if "x" in k else k
        assert L.xb_ssm_conv(C.byref(_conv(c, **k)), None) == ARG and b"overlap" in L.xb_last_error(), k
    states = dict(n_slots=3, state_in=AT)
    for at in (AT + 2, AT + 3 * 3 * 24 * 2 - 2, AT - 16):
        assert L.xb_ssm_conv(C.byref(_conv(c, state_out=at, **states)), None) == ARG and b"states overlap" in L.xb_last_error()
    for k in [dict(y=AT), dict(y=AT + row)] + [{n: AT + (1 << 20)} for n in ("delta", "B", "C")] + [dict(z=AT + (1 << 20) + row, ldz=24)]:
        assert L.xb_ssm_scan(C.byref(_scan(c, **k)), AT, 1 << 40, None) == ARG and b"overlap" in L.xb_last_error(), k
    assert L.xb_ssm_scan(C.byref(_scan(c, h_in=AT, h_out=AT + 4, n_slots=3)), AT, 1 << 40, None) == ARG and b"states overlap" in L.xb_last_error()
    for k in (dict(Y=AT), dict(Y=AT, y_dtype=c.XB_F32), dict(Y=AT + 62, N=32, ldy=32, stride_b=256), dict(Y=AT + 9 * 64, N=32, ldy=32, stride_b=256)):
        assert L.xb_lora_gemm(C.byref(_lora(c, **k)), AT, 1 << 40, None) == ARG and b"overlap" in L.xb_last_error(), k


def test_no_scratch_without_adapters():
    m = pkg.load()
    c, L = m.capi, m.lib()
    for dtype in (c.XB_F32, c.XB_BF16):
        for k in (dict(n_adapters=0), dict(r=0, ldb=0), dict(n_adapters=0, M=100_000), dict(n_adapters=0, M=700, ldx=33, K=33, ldw=33, lda=33)):
            assert L.xb_lora_workspace_bytes(C.byref(_lora(c, dtype=dtype, y_dtype=dtype, **k))) == 0, k


def test_scratch_goes_by_the_rows_and_not_by_the_table():
    m = pkg.load()
    c, L = m.capi, m.lib()
    for n in (1_000, 100_000, 10_000_000):
        for k in (dict(M=600, ldx=33, K=33, ldw=33, lda=33, stride_a=264), dict(M=2100, N=304, ldy=304, stride_b=304 * 8), dict(M=2100, N=304, ldy=304, stride_a=0),
                  dict(M=80_000, N=1024, ldy=1024, stride_b=0)):
            a = _lora(c, n_adapters=n, **k)
            named = min(n, a.M)
            most = a.M * 32 * 4 + a.M * 40 * 2 + a.N * 40 * 2 + max(32 << 20, named * (a.N * 32 * 4 + a.r * 40 * 2)) + 4 * (n + 1 + named) + 8 * 256
            assert 0 < L.xb_lora_workspace_bytes(C.byref(a)) <= most, (n, k)
            if k.get("stride_b") == 0:                         # one B for all: its room does not go by them at all
                assert L.xb_lora_workspace_bytes(C.byref(a)) <= a.M * 32 * 4 + a.N * 32 * 4 + 4 * 256


def test_the_module_of_another_torch_is_refused(monkeypatch):
    m = pkg.load()
    assert m.capi.tensors().torch_version == torch.__version__.split("+")[0]
    monkeypatch.setattr(m.capi, "_tensors", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(RuntimeError, match="build it again"):
        m.capi.tensors()


@pytest.mark.parametrize("suffix", ["", "+cu128", ".dev20260101+cu128", "a0+git1234567"])
def test_builds_of_one_torch_are_one(monkeypatch, suffix):
    m = pkg.load()
    monkeypatch.setattr(torch, "__version__", m.capi.tensors().torch_version + suffix)
    monkeypatch.setattr(m.capi, "_tensors", None)
    assert m.capi.tensors().torch_version
