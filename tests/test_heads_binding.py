"""What ops.qk_norm_rope, ops.linear_attention and ops.prefix_attention hand the C ABI, and which tensors they refuse. The C functions are Python
callbacks here and the tensors lie on the CPU, so nothing runs on a GPU."""
import ctypes as C

import pytest
import torch

import pkg

F16, I32 = torch.float16, torch.int32


@pytest.fixture
def bound(monkeypatch):
    pkg.load()
    from x_deeplearning_b200 import capi, ops
    m, seen, need = capi.tensors(), [], [0]

    def taken(kind):
        def f(a, *rest):
            seen.append(({n: getattr(a.contents, n) for n, _ in kind._fields_}, rest))
            return 0
        return f
    with_scratch = lambda kind: C.CFUNCTYPE(C.c_int, C.POINTER(kind), C.c_void_p, C.c_size_t, C.c_void_p)(taken(kind))
    bytes_ = C.CFUNCTYPE(C.c_size_t, C.c_void_p)
    fs = {"xb_qk_norm_rope": C.CFUNCTYPE(C.c_int, C.POINTER(capi.QkNormRopeArgs), C.c_void_p)(taken(capi.QkNormRopeArgs)),
          "xb_linear_attention": with_scratch(capi.LinearAttentionArgs), "xb_prefix_attention": with_scratch(capi.PrefixAttentionArgs),
          "xb_linear_attention_workspace_bytes": bytes_(lambda a: need[0]), "xb_prefix_attention_workspace_bytes": bytes_(lambda a: need[0])}
    real = {n: C.cast(getattr(capi.lib(), n), C.c_void_p).value for n in fs}
    for n, f in fs.items():
        m.bind(n, C.cast(f, C.c_void_p).value)
    monkeypatch.setattr(ops, "_where", lambda: (-1, 77))                    # a CPU tensor's device is -1
    yield ops, capi, seen, need
    for n, a in real.items():
        m.bind(n, a)


def _refused(seen, capi, name, call, good, cases):
    n = len(seen)
    for bad in cases:
        with pytest.raises(capi.XbError, match=name):
            call(**{**good, **bad})
    assert len(seen) == n


def test_rope(bound):
    ops, capi, seen, _ = bound
    y = torch.zeros(5, 8, 32, dtype=F16)
    q, k = y[:, :4], y[:, 4:6]
    pos, freqs, w = torch.zeros(5, dtype=I32), torch.zeros(8), torch.zeros(32)
    a, b = ops.qk_norm_rope(q, k, pos, freqs, q_weight=w, eps=0.5, adjacent=True, out_q=q)
    s, rest = seen[-1]
    assert rest == (77,) and a.data_ptr() == q.data_ptr() and b.shape == (5, 2, 32)
    assert (s["q"], s["q_row"], s["q_head"], s["k"], s["k_row"], s["yq"], s["yq_row"], s["yk"], s["yk_row"], s["yk_head"]) == (
        q.data_ptr(), 256, 32, k.data_ptr(), 256, q.data_ptr(), 256, b.data_ptr(), 64, 32)
    assert (s["q_weight"], s["k_weight"], s["positions"], s["freqs"], s["rows"], s["Hq"], s["Hk"], s["d"], s["rot"], s["norm"], s["adjacent"], s["eps"],
            s["dtype"]) == (w.data_ptr(), None, pos.data_ptr(), freqs.data_ptr(), 5, 4, 2, 32, 16, 1, 1, 0.5, capi.XB_F16)
    assert ops.qk_norm_rope(q, None, None, None)[1] is None and (seen[-1][0]["Hk"], seen[-1][0]["rot"]) == (0, 0)
    _refused(seen, capi, "qk_norm_rope", ops.qk_norm_rope, dict(q=q, k=k, positions=pos, freqs=freqs), (
        dict(q=q[0]), dict(q=y[:, :4, ::2]), dict(q=q.double()), dict(k=k[:4]), dict(k=k.float()), dict(k=k[..., :16]), dict(k=k[0]), dict(positions=pos.long()),
        dict(positions=pos[:4]), dict(positions=None), dict(freqs=freqs.half()), dict(freqs=freqs[::2]), dict(freqs=torch.zeros(33)), dict(q_weight=w[:31]),
        dict(k_weight=w.half()), dict(k=None, k_weight=w), dict(k=None, out_k=k), dict(out_q=torch.zeros(5, 4, 32)), dict(out_q=q[:4])))


def test_linear(bound):
    ops, capi, seen, need = bound
    q, k, v = torch.zeros(12, 4, 16, dtype=F16), torch.zeros(12, 2, 16, dtype=F16), torch.zeros(12, 2, 24, dtype=F16)
    ld, h, slots = torch.zeros(4), torch.zeros(7, 4, 16, 24), torch.zeros(3, dtype=I32)
    off = torch.zeros(6, dtype=I32)
    need[0] = 100
    y = ops.linear_attention(q, k, v, ld, scale=0.25, T=4, longest=4, h_in=h, h_out=h, slots=slots)
    s, rest = seen[-1]
    assert y.shape == (12, 4, 24) and y.dtype == F16 and rest[0] and rest[1] >= 100 and rest[2] == 77
    assert (s["q"], s["q_row"], s["q_head"], s["k_row"], s["v_row"], s["v_head"], s["y"], s["y_row"], s["y_head"], s["log_decay"], s["offsets"]) == (
        q.data_ptr(), 64, 16, 32, 48, 24, y.data_ptr(), 96, 24, ld.data_ptr(), None)
    assert (s["slots"], s["h_in"], s["h_out"], s["rows"], s["longest"], s["batch"], s["n_slots"], s["H"], s["Hkv"], s["dk"], s["dv"], s["scale"], s["dtype"]) == (
        slots.data_ptr(), h.data_ptr(), h.data_ptr(), 12, 4, 3, 7, 4, 2, 16, 24, 0.25, capi.XB_F16)
    ops.linear_attention(q, k, v, ld, offsets=off)
    assert (seen[-1][0]["offsets"], seen[-1][0]["batch"], seen[-1][0]["n_slots"]) == (off.data_ptr(), 5, 0)
    _refused(seen, capi, "linear_attention", ops.linear_attention, dict(q=q, k=k, v=v, log_decay=ld, T=4), (
        dict(q=q[0]), dict(k=k[:11]), dict(k=k.float()), dict(k=k[..., :8]), dict(v=v[..., ::2]), dict(v=v[:, :1]), dict(log_decay=ld[:3]), dict(log_decay=ld.half()),
        dict(T=5), dict(T=0), dict(T=None, offsets=off.long()), dict(T=None, offsets=off[:0]), dict(slots=slots[:2]), dict(slots=slots.long()), dict(h_in=h[:, :3]),
        dict(h_in=h.half()), dict(h_in=h[..., :23]), dict(h_in=h.transpose(2, 3)), dict(h_in=h, h_out=h[:6]), dict(h_in=h[0]), dict(out=torch.zeros(12, 4, 24)),
        dict(out=torch.zeros(11, 4, 24, dtype=F16)), dict(workspace=torch.zeros(4000, dtype=torch.uint8)[::2])))


def test_prefix(bound):
    ops, capi, seen, need = bound
    q, k, v = torch.zeros(12, 4, 64, dtype=F16), torch.zeros(30, 2, 64, dtype=F16), torch.zeros(30, 2, 64, dtype=F16)
    pk, pv = torch.zeros(50, 2, 64, dtype=F16), torch.zeros(50, 2, 64, dtype=F16)
    own, pre, mem = torch.zeros(13, dtype=I32), torch.zeros(4, dtype=I32), torch.zeros(4, dtype=I32)
    need[0] = 100
    y = ops.prefix_attention(q, k, v, T=1, own_offsets=own, prefix_k=pk, prefix_v=pv, prefix_offsets=pre, members=mem, scale=0.5)
    s, rest = seen[-1]
    assert y.shape == (12, 4, 64) and rest[0] and rest[1] >= 100 and rest[2] == 77
    assert (s["q"], s["k"], s["v"], s["prefix_k"], s["prefix_v"], s["own_offsets"], s["prefix_offsets"], s["members"], s["offsets"]) == (
        q.data_ptr(), k.data_ptr(), v.data_ptr(), pk.data_ptr(), pv.data_ptr(), own.data_ptr(), pre.data_ptr(), mem.data_ptr(), None)
    assert (s["rows"], s["own_rows"], s["prefix_rows"], s["batch"], s["prefixes"], s["H"], s["Hkv"], s["d"], s["scale"], s["dtype"]) == (
        12, 30, 50, 12, 3, 4, 2, 64, 0.5, capi.XB_F16)
    ops.prefix_attention(q, T=3, prefix_k=pk, prefix_v=pv)
    assert (seen[-1][0]["k"], seen[-1][0]["own_rows"], seen[-1][0]["prefixes"], seen[-1][0]["batch"]) == (None, 0, 1, 4)
    _refused(seen, capi, "prefix_attention", ops.prefix_attention, dict(q=q, k=k, v=v, T=1, own_offsets=own, prefix_k=pk, prefix_v=pv, prefix_offsets=pre, members=mem), (
        dict(q=q[0]), dict(q=q[..., ::2]), dict(k=k.float()), dict(k=None), dict(v=None), dict(v=v[:29]), dict(k=k[:, :1]), dict(k=None, v=None), dict(prefix_k=None),
        dict(prefix_k=None, prefix_v=None), dict(prefix_v=pv[..., :32]), dict(prefix_v=pv[:49]), dict(own_offsets=own[:12]), dict(own_offsets=own.long()),
        dict(prefix_offsets=pre[:3]), dict(prefix_offsets=pre[:0], members=None), dict(members=mem[::2]), dict(members=mem.long()), dict(T=5),
        dict(T=None, offsets=own[:5].long()), dict(out=torch.zeros(12, 4, 64)), dict(out=torch.zeros(12, 4, 32, dtype=F16)),
        dict(workspace=torch.zeros(4000, dtype=torch.uint8)[::2])))
