"""What the attention over lists refuses, and its scratch sizes: host logic alone, on addresses that nothing reads."""
import ctypes as C

import pkg

AT, FAR = 1 << 20, 1 << 30
ARG, UNSUPPORTED, SCRATCH, LIMIT = -1, -2, -4, -5


def _with(a, k):
    for n, v in k.items():
        setattr(a, n, v)
    return a


def _rope(c, **k):
    a = c.QkNormRopeArgs()
    a.q, a.k, a.yq, a.yk, a.positions, a.freqs = AT, AT + 1024, FAR, 2 * FAR, AT, AT
    a.rows, a.Hq, a.Hk, a.d, a.rot, a.norm, a.eps, a.dtype = 10, 4, 2, 32, 32, 1, 1e-6, c.XB_F16
    a.q_row = a.k_row = 4096
    a.q_head = a.k_head = a.yq_head = a.yk_head = 32
    a.yq_row, a.yk_row = 128, 64
    return _with(a, k)


def test_rope():
    m = pkg.load()
    c, L = m.capi, m.lib()
    assert L.xb_qk_norm_rope(None, None) == ARG
    for rc, k in ((UNSUPPORTED, dict(dtype=c.XB_I32)), (ARG, dict(rows=-1)), (ARG, dict(Hq=-1)), (ARG, dict(d=0)), (ARG, dict(rot=31)), (ARG, dict(rot=34)),
                  (LIMIT, dict(d=257)), (LIMIT, dict(rows=1 << 31)), (LIMIT, dict(Hk=65536)), (ARG, dict(eps=-1.0)), (ARG, dict(eps=float("nan"))),
                  (ARG, dict(norm=0, q_weight=AT)), (ARG, dict(q=None)), (ARG, dict(yk=None)), (ARG, dict(positions=None)), (ARG, dict(freqs=None)),
                  (ARG, dict(q_row=-1)), (ARG, dict(yq_row=127)), (ARG, dict(yq_head=31)), (ARG, dict(yq=AT)), (ARG, dict(yq=AT + 2, yq_row=4096)),
                  (ARG, dict(yk=AT + 128, yk_row=4096)), (ARG, dict(yk=FAR)), (ARG, dict(yq=AT + 64, yq_row=4096))):
        assert L.xb_qk_norm_rope(C.byref(_rope(c, **k)), None) == rc, k
        assert b"xb_qk_norm_rope" in L.xb_last_error()
    assert L.xb_qk_norm_rope(C.byref(_rope(c, rows=0, q=None)), None) == 0
    assert L.xb_qk_norm_rope(C.byref(_rope(c, Hq=0, Hk=0)), None) == 0


def _linear(c, **k):
    a = c.LinearAttentionArgs()
    a.q, a.k, a.v, a.y, a.log_decay = AT, AT, AT, FAR, AT
    a.rows, a.batch, a.H, a.Hkv, a.dk, a.dv, a.scale, a.dtype = 12, 3, 4, 2, 16, 24, 1.0, c.XB_BF16
    a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head, a.y_row, a.y_head = 64, 16, 32, 16, 48, 24, 96, 24
    return _with(a, k)


def test_linear():
    m = pkg.load()
    c, L = m.capi, m.lib()
    assert L.xb_linear_attention(None, None, 0, None) == ARG and L.xb_linear_attention_workspace_bytes(None) == 0
    for rc, k in ((UNSUPPORTED, dict(dtype=c.XB_I32)), (ARG, dict(H=0)), (ARG, dict(Hkv=3)), (ARG, dict(dk=0)), (ARG, dict(dv=0)), (LIMIT, dict(dk=129)),
                  (LIMIT, dict(dv=129)), (LIMIT, dict(H=65536)), (ARG, dict(batch=5)), (ARG, dict(batch=-1)), (ARG, dict(rows=-1)), (ARG, dict(longest=-1)),
                  (LIMIT, dict(batch=2**31 - 1, offsets=AT)), (LIMIT, dict(rows=1 << 31, batch=1)), (ARG, dict(h_in=AT, n_slots=2)),
                  (ARG, dict(h_out=AT, n_slots=-1, slots=AT)), (ARG, dict(log_decay=None)), (ARG, dict(v=None)), (ARG, dict(y=None)), (ARG, dict(k_head=-1)),
                  (ARG, dict(y_row=95)), (ARG, dict(y=AT)), (ARG, dict(q=FAR + 16)), (ARG, dict(h_in=AT, h_out=AT + 4, n_slots=3))):
        assert L.xb_linear_attention(C.byref(_linear(c, **k)), None, 0, None) == rc, k
        assert b"xb_linear_attention" in L.xb_last_error()
    assert L.xb_linear_attention(C.byref(_linear(c, rows=0, batch=0, q=None)), None, 0, None) == 0
    # scratch: none for short lists; long ones that are cut keep a state (with states to begin with, two) for every piece but the last
    bytes_ = lambda **k: L.xb_linear_attention_workspace_bytes(C.byref(_linear(c, **k)))
    assert bytes_() == 0 and bytes_(rows=-1) == 0
    long = dict(rows=100_000, batch=1)
    need = bytes_(**long)
    assert need > 0 and bytes_(h_in=AT, n_slots=1, **long) == 2 * need
    assert L.xb_linear_attention(C.byref(_linear(c, **long)), AT, need - 1, None) == SCRATCH
    assert L.xb_linear_attention(C.byref(_linear(c, **long)), None, need, None) == SCRATCH
    assert L.xb_linear_attention(C.byref(_linear(c, **long)), AT + 4, need, None) == ARG


def _prefix(c, **k):
    a = c.PrefixAttentionArgs()
    a.q, a.k, a.v, a.prefix_k, a.prefix_v, a.y = AT, AT, AT, AT, AT, FAR
    a.rows, a.own_rows, a.prefix_rows, a.batch, a.prefixes, a.H, a.Hkv, a.d, a.scale, a.dtype = 12, 12, 40, 4, 2, 4, 2, 64, 0.125, c.XB_BF16
    a.q_row, a.y_row, a.k_row, a.v_row, a.prefix_k_row, a.prefix_v_row = 256, 256, 128, 128, 128, 128
    a.q_head = a.k_head = a.v_head = a.prefix_k_head = a.prefix_v_head = a.y_head = 64
    return _with(a, k)


def test_prefix():
    m = pkg.load()
    c, L = m.capi, m.lib()
    assert L.xb_prefix_attention(None, None, 0, None) == ARG and L.xb_prefix_attention_workspace_bytes(None) == 0
    for rc, k in ((UNSUPPORTED, dict(dtype=c.XB_F32)), (ARG, dict(H=0)), (ARG, dict(Hkv=3)), (ARG, dict(d=0)), (UNSUPPORTED, dict(d=60)), (LIMIT, dict(d=136)),
                  (LIMIT, dict(H=258)), (LIMIT, dict(H=65536, Hkv=65536)), (ARG, dict(rows=-1)), (ARG, dict(prefixes=-1)), (ARG, dict(own_rows=-1)),
                  (LIMIT, dict(batch=2**31 - 1)), (LIMIT, dict(rows=1 << 31)), (LIMIT, dict(prefix_rows=1 << 31)), (ARG, dict(scale=0.0)), (ARG, dict(scale=-1.0)),
                  (ARG, dict(scale=float("nan"))), (ARG, dict(scale=float("inf"))), (ARG, dict(batch=5)), (ARG, dict(k=None)), (ARG, dict(v=None)),
                  (ARG, dict(k=None, v=None)), (ARG, dict(prefix_v=None)), (ARG, dict(q=None)), (ARG, dict(y=None)), (ARG, dict(own_rows=11)), (ARG, dict(prefixes=0)),
                  (ARG, dict(prefixes=3)), (ARG, dict(prefix_rows=41)), (UNSUPPORTED, dict(q=AT + 2)), (UNSUPPORTED, dict(prefix_k=AT + 8)),
                  (UNSUPPORTED, dict(k_row=132)), (UNSUPPORTED, dict(v_head=63)), (UNSUPPORTED, dict(prefix_v_row=56)), (UNSUPPORTED, dict(q_head=0)),
                  (LIMIT, dict(k_row=1 << 39)), (ARG, dict(y_row=-1))):
        assert L.xb_prefix_attention(C.byref(_prefix(c, **k)), None, 0, None) == rc, k
        assert b"xb_prefix_attention" in L.xb_last_error()
        assert L.xb_prefix_attention_workspace_bytes(C.byref(_prefix(c, **k))) == 0
    need = L.xb_prefix_attention_workspace_bytes(C.byref(_prefix(c)))
    assert need > 0
    for rc, k, ws, n in ((SCRATCH, {}, AT, need - 1), (SCRATCH, {}, None, need), (ARG, {}, AT + 8, need), (ARG, dict(y=AT), AT, need), (ARG, dict(y_row=255), AT, need),
                         (ARG, dict(y_head=63), AT, need), (ARG, dict(prefix_v=FAR + 256), AT, need), (ARG, dict(k=FAR + 16 * 64), AT, need)):
        assert L.xb_prefix_attention(C.byref(_prefix(c, **k)), ws, n, None) == rc, k
    assert L.xb_prefix_attention(C.byref(_prefix(c, batch=0, rows=0, q=None)), None, 0, None) == 0
