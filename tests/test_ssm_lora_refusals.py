"""What xb_ssm_conv, xb_ssm_scan and xb_lora_gemm refuse, and their scratch sizes: host logic alone, on addresses that nothing reads."""
import ctypes as C

import pytest

import pkg

AT = 4096


def _conv(c, **k):
    a = c.SsmConvArgs()
    a.x = a.y = a.w = AT
    a.rows, a.batch, a.D, a.K, a.dtype, a.ldx, a.ldy = 12, 3, 24, 4, c.XB_F16, 24, 24
    for n, v in k.items():
        setattr(a, n, v)
    return a


def _scan(c, **k):
    a = c.SsmScanArgs()
    a.x = a.delta = a.B = a.C = a.y = a.A = AT
    a.rows, a.batch, a.D, a.N, a.groups, a.dtype = 12, 3, 24, 16, 2, c.XB_BF16
    a.ldx = a.lddelta = a.ldy = 24
    a.ldb = a.ldc = 32
    for n, v in k.items():
        setattr(a, n, v)
    return a


def _lora(c, **k):
    a = c.LoraArgs()
    a.X = a.W = a.A = a.B = a.adapter = a.Y = AT
    a.M, a.N, a.K, a.r, a.n_adapters, a.trans_w, a.dtype, a.y_dtype = 10, 16, 32, 8, 3, 1, c.XB_F16, c.XB_F16
    a.ldx = a.ldw = a.lda = 32
    a.ldy, a.ldb, a.stride_a, a.stride_b = 16, 8, 256, 128
    for n, v in k.items():
        setattr(a, n, v)
    return a


ARG, UNSUPPORTED, SCRATCH, LIMIT = -1, -2, -4, -5


def test_conv():
    m = pkg.load()
    c, L = m.capi, m.lib()
    assert L.xb_ssm_conv(None, None) == ARG
    for rc, k in ((UNSUPPORTED, dict(dtype=c.XB_I32)), (ARG, dict(D=0)), (LIMIT, dict(K=1)), (LIMIT, dict(K=9)), (ARG, dict(batch=5)),
                  (ARG, dict(batch=-1)), (ARG, dict(rows=-1)), (LIMIT, dict(rows=1 << 31, batch=1)), (ARG, dict(state_in=AT, n_slots=2)),
                  (ARG, dict(state_out=AT, n_slots=-1, slots=AT)), (ARG, dict(w=None)), (ARG, dict(x=None)), (ARG, dict(y=None)),
                  (ARG, dict(ldx=23)), (ARG, dict(ldy=23))):
        assert L.xb_ssm_conv(C.byref(_conv(c, **k)), None) == rc, k
        assert b"xb_ssm_conv" in L.xb_last_error()
    assert L.xb_ssm_conv(C.byref(_conv(c, batch=0, rows=0, x=None)), None) == 0


def test_scan():
    m = pkg.load()
    c, L = m.capi, m.lib()
    assert L.xb_ssm_scan(None, None, 0, None) == ARG and L.xb_ssm_scan_workspace_bytes(None) == 0
    for rc, k in ((UNSUPPORTED, dict(dtype=c.XB_I64)), (ARG, dict(D=0)), (ARG, dict(N=0)), (LIMIT, dict(N=65, ldb=130, ldc=130)), (ARG, dict(groups=5)),
                  (ARG, dict(groups=0)), (ARG, dict(longest=-1)), (ARG, dict(batch=7)), (LIMIT, dict(rows=1 << 31, batch=1)),
                  (ARG, dict(h_in=AT, n_slots=2)), (ARG, dict(A=None)), (ARG, dict(x=None)), (ARG, dict(delta=None)), (ARG, dict(B=None)),
                  (ARG, dict(C=None)), (ARG, dict(y=None)), (ARG, dict(ldx=23)), (ARG, dict(lddelta=23)), (ARG, dict(ldy=23)),
                  (ARG, dict(z=AT, ldz=23)), (ARG, dict(ldb=31)), (ARG, dict(ldc=31))):
        assert L.xb_ssm_scan(C.byref(_scan(c, **k)), None, 0, None) == rc, k
        assert b"xb_ssm_scan" in L.xb_last_error()
    assert L.xb_ssm_scan(C.byref(_scan(c, batch=0, rows=0, x=None)), None, 0, None) == 0


def test_lora():
    m = pkg.load()
    c, L = m.capi, m.lib()
    assert L.xb_lora_gemm(None, None, 0, None) == ARG and L.xb_lora_workspace_bytes(None) == 0
    for rc, k in ((UNSUPPORTED, dict(dtype=c.XB_I32)), (UNSUPPORTED, dict(y_dtype=c.XB_BF16)), (ARG, dict(M=-1)), (ARG, dict(K=0)), (ARG, dict(r=-1)),
                  (LIMIT, dict(r=129, ldb=129)), (LIMIT, dict(M=(1 << 31) - 1000)), (LIMIT, dict(N=(1 << 31) - 1, ldy=1 << 31)),
                  (LIMIT, dict(K=(1 << 31) - 1, ldx=1 << 31, ldw=1 << 31, lda=1 << 31)), (ARG, dict(X=None)), (ARG, dict(W=None)), (ARG, dict(Y=None)), (ARG, dict(A=None)), (ARG, dict(B=None)),
                  (ARG, dict(adapter=None)), (ARG, dict(ldx=31)), (ARG, dict(ldw=31)), (ARG, dict(trans_w=0, ldw=15)), (ARG, dict(ldy=15)),
                  (ARG, dict(lda=31)), (ARG, dict(ldb=7)), (ARG, dict(stride_a=-1)), (ARG, dict(stride_b=-8))):
        assert L.xb_lora_gemm(C.byref(_lora(c, **k)), AT, 1 << 40, None) == rc, k
        assert b"xb_lora_gemm" in L.xb_last_error()
    assert L.xb_lora_gemm(C.byref(_lora(c, M=0)), None, 0, None) == 0
    assert L.xb_lora_gemm(C.byref(_lora(c, N=0)), None, 0, None) == 0


@pytest.mark.parametrize("M,N", [(1, 8), (64, 1024), (80000, 1024), (100, 100000)])
def test_lora_scratch(M, N):
    m = pkg.load()
    c, L = m.capi, m.lib()
    a = _lora(c, M=M, N=N, ldy=N, dtype=c.XB_F32, y_dtype=c.XB_F32)
    need = L.xb_lora_workspace_bytes(C.byref(a))
    assert 0 < need <= (128 << 20)
    assert L.xb_lora_gemm(C.byref(a), AT, need - 1, None) == SCRATCH
    assert L.xb_lora_gemm(C.byref(a), None, need, None) == SCRATCH
    assert L.xb_lora_gemm(C.byref(a), AT + 8, need, None) == ARG
