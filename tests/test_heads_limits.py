"""Sizes of xb_prefix_attention past what its plan counts in 32 bits are refused by name, and have no scratch size (host logic alone)."""
import ctypes as C

import pkg

AT, FAR = 1 << 20, 1 << 30
LIMIT = -5


def test_prefix():
    m = pkg.load()
    c, L = m.capi, m.lib()
    rows = 2**31 - 1024

    def call(**k):
        a = c.PrefixAttentionArgs()
        a.q, a.prefix_k, a.prefix_v, a.y, a.offsets, a.members, a.prefix_offsets = AT, AT, AT, FAR, AT, AT, AT
        a.rows, a.prefix_rows, a.batch, a.prefixes, a.H, a.Hkv, a.d, a.scale, a.dtype = rows, 40, 1 << 20, 2, 1, 1, 8, 1.0, c.XB_BF16
        a.q_row, a.y_row, a.prefix_k_row, a.prefix_v_row = 8, 1024, 8, 8
        a.q_head = a.prefix_k_head = a.prefix_v_head = a.y_head = 8
        for n, v in k.items():
            setattr(a, n, v)
        return C.byref(a)

    for k in (dict(prefixes=2**31 - 3000), dict(prefixes=2**31 - 2047, rows=10), dict(prefixes=2**31 - 1024, rows=10), dict(H=128, prefixes=2**31 - 3000),
              dict(H=128, prefixes=1 << 30, rows=rows - 8)):
        assert L.xb_prefix_attention_workspace_bytes(call(**k)) == 0, k
        assert L.xb_prefix_attention(call(**k), AT, 1 << 40, None) == LIMIT, k
        assert b"xb_prefix_attention" in L.xb_last_error()
    # as many items as are counted: their scratch is what it is
    assert 64 * 2**30 < L.xb_prefix_attention_workspace_bytes(call(H=128, prefixes=1 << 20)) < 1 << 40
    assert 32 * 2**30 < L.xb_prefix_attention_workspace_bytes(call(prefixes=2**31 - 2048, rows=10)) < 1 << 40
