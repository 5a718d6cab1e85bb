"""Inputs and outputs of one row that share memory: refused by where they begin and end, whatever the row strides say (host logic alone, on addresses
that nothing reads)."""
import ctypes as C

import pytest

import pkg

AT, FAR = 1 << 20, 1 << 30
ARG = -1


def _one_row(a, **k):
    a.rows = 1
    for n, v in k.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("stride", [0, 1, 4, 128])
def test_rope(stride):
    m = pkg.load()
    c, L = m.capi, m.lib()
    for at in (AT - 64, AT - 2, AT + 2, AT + 64, AT + 254):
        a = _one_row(c.QkNormRopeArgs(), q=AT, yq=at, q_head=32, yq_head=32, q_row=stride, yq_row=stride, Hq=4, d=32, norm=1, eps=1e-6, dtype=c.XB_F16)
        assert L.xb_qk_norm_rope(C.byref(a), None) == ARG and b"overlap" in L.xb_last_error()
        a = _one_row(c.QkNormRopeArgs(), q=AT, yq=FAR, k=AT, yk=FAR + at - AT, q_head=32, yq_head=32, k_head=32, yk_head=32, yq_row=stride, yk_row=stride, Hq=4, Hk=4, d=32,
                     norm=1, eps=1e-6, dtype=c.XB_F16)
        assert L.xb_qk_norm_rope(C.byref(a), None) == ARG and b"overlap" in L.xb_last_error()


@pytest.mark.parametrize("stride", [0, 1, 4, 128])
def test_linear(stride):
    m = pkg.load()
    c, L = m.capi, m.lib()
    for which in ("q", "k", "v"):
        for at in (AT - 64, AT - 2, AT + 2, AT + 64, AT + 254):
            a = _one_row(c.LinearAttentionArgs(), q=FAR, k=FAR, v=FAR, log_decay=FAR, y=AT, batch=1, H=4, Hkv=4, dk=32, dv=32, scale=1.0, dtype=c.XB_BF16,
                         q_head=32, k_head=32, v_head=32, y_head=32, q_row=stride, k_row=stride, v_row=stride, y_row=stride)
            setattr(a, which, at)
            assert L.xb_linear_attention(C.byref(a), None, 0, None) == ARG and b"overlap" in L.xb_last_error()


@pytest.mark.parametrize("stride", [0, 8, 128])
def test_prefix(stride):
    m = pkg.load()
    c, L = m.capi, m.lib()
    for which in ("q", "k", "v"):
        for at in (AT - 64, AT - 16, AT + 16, AT + 64, AT + 240):
            a = _one_row(c.PrefixAttentionArgs(), q=FAR, k=FAR, v=FAR, y=AT, own_rows=1, batch=1, H=4, Hkv=4, d=32, scale=1.0, dtype=c.XB_BF16,
                         q_head=32, k_head=32, v_head=32, y_head=32, q_row=stride, k_row=stride, v_row=stride, y_row=stride)
            setattr(a, which, at)
            assert L.xb_prefix_attention(C.byref(a), 1 << 40, 1 << 40, None) == ARG and b"overlap" in L.xb_last_error()
