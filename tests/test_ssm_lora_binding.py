"""What ops.ssm_conv, ops.ssm_scan and ops.lora_gemm hand the C ABI, and which tensors they refuse. The C functions are Python callbacks
here and the tensors lie on the CPU, so nothing runs on a GPU."""
import ctypes as C

import pytest
import torch

import pkg


@pytest.fixture
def bound(monkeypatch):
    pkg.load()
    from x_deeplearning_b200 import capi, ops
    m, seen, need, result = capi.tensors(), [], [0], [0]

    def taken(kind):
        def f(a, *rest):
            seen.append(({n: getattr(a.contents, n) for n, _ in kind._fields_}, rest))
            return result[0]
        return f
    fs = {"xb_ssm_conv": C.CFUNCTYPE(C.c_int, C.POINTER(capi.SsmConvArgs), C.c_void_p)(taken(capi.SsmConvArgs)),
          "xb_ssm_scan": C.CFUNCTYPE(C.c_int, C.POINTER(capi.SsmScanArgs), C.c_void_p, C.c_size_t, C.c_void_p)(taken(capi.SsmScanArgs)),
          "xb_lora_gemm": C.CFUNCTYPE(C.c_int, C.POINTER(capi.LoraArgs), C.c_void_p, C.c_size_t, C.c_void_p)(taken(capi.LoraArgs)),
          "xb_ssm_scan_workspace_bytes": C.CFUNCTYPE(C.c_size_t, C.c_void_p)(lambda a: need[0]),
          "xb_lora_workspace_bytes": C.CFUNCTYPE(C.c_size_t, C.c_void_p)(lambda a: need[0])}
    real = {n: C.cast(getattr(capi.lib(), n), C.c_void_p).value for n in fs}
    for n, f in fs.items():
        m.bind(n, C.cast(f, C.c_void_p).value)
    monkeypatch.setattr(ops, "_where", lambda: (-1, 77))                    # a CPU tensor's device is -1
    yield ops, capi, seen, need, result
    for n, a in real.items():
        m.bind(n, a)


def test_conv(bound):
    ops, capi, seen, _, result = bound
    x, w, b = torch.zeros(12, 30, dtype=torch.float16)[:, :24], torch.zeros(24, 4, dtype=torch.float16), torch.zeros(24, dtype=torch.float16)
    st, slots = torch.zeros(7, 3, 24, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    y = ops.ssm_conv(x, w, b, T=4, state_in=st, state_out=st, slots=slots, silu=False)
    a, rest = seen[-1]
    assert rest == (77,) and y.shape == (12, 24) and y.dtype == torch.float16
    assert (a["x"], a["ldx"], a["y"], a["ldy"], a["w"], a["bias"], a["offsets"], a["slots"]) == (
        x.data_ptr(), 30, y.data_ptr(), 24, w.data_ptr(), b.data_ptr(), None, slots.data_ptr())
    assert (a["state_in"], a["state_out"], a["rows"], a["batch"], a["n_slots"], a["D"], a["K"], a["silu"], a["dtype"]) == (
        st.data_ptr(), st.data_ptr(), 12, 3, 7, 24, 4, 0, capi.XB_F16)
    off = torch.zeros(6, dtype=torch.int32)
    ops.ssm_conv(x, w, offsets=off)
    a, _ = seen[-1]
    assert (a["offsets"], a["batch"], a["bias"], a["state_in"], a["n_slots"], a["silu"]) == (off.data_ptr(), 5, None, None, 0, 1)
    ops.ssm_conv(x[:1], w)
    assert (seen[-1][0]["batch"], seen[-1][0]["rows"]) == (1, 1)
    n = len(seen)
    for bad in (dict(x=x.t()), dict(x=x.float()), dict(w=w[:, ::2]), dict(w=w[:23]), dict(bias=b[:23]), dict(T=5), dict(T=0), dict(T=-1),
                dict(offsets=off.long()), dict(offsets=off[:0]), dict(offsets=torch.zeros(12, dtype=torch.int32)[::2]), dict(state_in=st[:, :2]), dict(state_in=st.float()),
                dict(state_in=st, state_out=st[:6]), dict(T=4, slots=slots[:2]), dict(T=4, slots=slots.float()), dict(out=torch.zeros(12, 24)),
                dict(out=torch.zeros(11, 24, dtype=torch.float16))):
        with pytest.raises(capi.XbError, match="ssm_conv"):
            ops.ssm_conv(**{**dict(x=x, w=w), **bad})
    assert len(seen) == n
    result[0] = -1
    with pytest.raises(capi.XbError):
        ops.ssm_conv(x, w)


def test_scan(bound):
    ops, capi, seen, need, result = bound
    bf = torch.bfloat16
    x, d, z = (torch.zeros(12, w, dtype=bf)[:, :24] for w in (24, 32, 40))
    B, C_ = torch.zeros(12, 32, dtype=bf), torch.zeros(12, 48, dtype=bf)[:, :32]
    A, D, b, h = torch.zeros(24, 16), torch.zeros(24), torch.zeros(24), torch.zeros(3, 24, 16)
    h2 = torch.zeros(3, 24, 16)
    y = ops.ssm_scan(x, d, A, B, C_, D=D, z=z, delta_bias=b, groups=2, T=6, h_in=h, h_out=h2)
    a, rest = seen[-1]
    assert rest == (None, 0, 77) and y.shape == (12, 24)
    assert [a[k] for k in ("x", "delta", "z", "B", "C", "y", "A", "skip", "delta_bias", "h_in", "h_out")] == [
        t.data_ptr() for t in (x, d, z, B, C_, y, A, D, b, h, h2)]
    assert [a[k] for k in ("ldx", "lddelta", "ldz", "ldb", "ldc", "ldy")] == [24, 32, 40, 32, 48, 24]
    assert [a[k] for k in ("rows", "longest", "batch", "n_slots", "D", "N", "groups", "softplus", "dtype", "offsets", "slots")] == [
        12, 0, 2, 3, 24, 16, 2, 1, capi.XB_BF16, None, None]
    # scratch: the call's own, or the caller's
    need[0] = 1000
    ops.ssm_scan(x, d, A, B, C_, groups=2, softplus=False, longest=9)
    a, rest = seen[-1]
    assert rest[0] and rest[1] == 1000 and (a["longest"], a["softplus"], a["z"], a["ldz"], a["h_in"]) == (9, 0, None, 0, None)
    ws = torch.zeros(2000, dtype=torch.uint8)
    ops.ssm_scan(x, d, A, B, C_, groups=2, workspace=ws)
    assert seen[-1][1] == (ws.data_ptr(), 2000, 77)
    n = len(seen)
    for bad in (dict(delta=d[:11]), dict(delta=d.half()), dict(A=A.half()), dict(A=A[:23]), dict(A=torch.zeros(16, 24).t()), dict(B=B[:, :31]),
                dict(C=C_.float()), dict(D=D[:23]), dict(D=D.half()), dict(z=z[:, :23]), dict(delta_bias=b.half()), dict(groups=0), dict(groups=3),
                dict(h_in=h.half()), dict(h_in=h[:, :, :15]), dict(h_in=h, h_out=h2[:2]), dict(slots=torch.zeros(2, dtype=torch.int32)), dict(T=7),
                dict(workspace=torch.zeros(4000, dtype=torch.uint8)[::2]), dict(out=torch.zeros(12, 25, dtype=bf))):
        with pytest.raises(capi.XbError, match="ssm_scan"):
            ops.ssm_scan(**{**dict(x=x, delta=d, A=A, B=B, C=C_, groups=2), **bad})
    with pytest.raises((AttributeError, TypeError)):
        ops.ssm_scan(x, None, A, B, 3)
    assert len(seen) == n


def test_lora(bound):
    ops, capi, seen, need, result = bound
    h = torch.float16
    X, W = torch.zeros(10, 40, dtype=h)[:, :32], torch.zeros(16, 32, dtype=h)
    A, B, ad = torch.zeros(3, 8, 40, dtype=h)[:, :, :32], torch.zeros(3, 16, 8, dtype=h), torch.zeros(10, dtype=torch.int32)
    bias, scale = torch.zeros(16), torch.zeros(3)
    need[0] = 512
    Y = ops.lora_gemm(X, W, A, B, ad, bias=bias, scale=scale, trans_b=True, out_dtype=torch.float32)
    a, rest = seen[-1]
    assert rest[0] and rest[1:] == (512, 77) and Y.dtype == torch.float32 and Y.shape == (10, 16)
    assert [a[k] for k in ("M", "N", "K", "r", "n_adapters", "trans_w", "dtype", "y_dtype")] == [10, 16, 32, 8, 3, 1, capi.XB_F16, capi.XB_F32]
    assert [a[k] for k in ("X", "W", "A", "B", "scale", "bias", "adapter", "Y")] == [t.data_ptr() for t in (X, W, A, B, scale, bias, ad, Y)]
    assert [a[k] for k in ("ldx", "ldw", "lda", "stride_a", "ldb", "stride_b", "ldy")] == [40, 32, 40, 320, 8, 128, 16]
    Y = ops.lora_gemm(X, W.t().contiguous(), A, B, ad)
    assert Y.dtype == h and (seen[-1][0]["ldw"], seen[-1][0]["trans_w"], seen[-1][0]["scale"], seen[-1][0]["bias"]) == (16, 0, None, None)
    n = len(seen)
    for bad in (dict(X=X.t()), dict(W=W[:, :31]), dict(W=W.float()), dict(A=A[:2]), dict(A=A[:, :, ::2]), dict(A=A[0]), dict(B=B[:, :15]),
                dict(B=B.float()), dict(adapter=ad.long()), dict(adapter=ad[:9]), dict(bias=bias[:15]), dict(bias=bias.half()), dict(scale=scale[:2]),
                dict(Y=torch.zeros(10, 15, dtype=h)), dict(workspace=torch.zeros(10, 10, dtype=torch.uint8))):
        with pytest.raises(capi.XbError, match="lora_gemm"):
            ops.lora_gemm(**{**dict(X=X, W=W, A=A, B=B, adapter=ad, trans_b=True), **bad})
    assert len(seen) == n


def test_tensors_of_another_device(bound, monkeypatch):
    ops, capi, seen, _, _ = bound
    monkeypatch.setattr(ops, "_where", lambda: (0, 77))
    with pytest.raises(capi.XbError, match="on device -1"):
        ops.ssm_conv(torch.zeros(4, 8), torch.zeros(8, 4))
    assert not seen
