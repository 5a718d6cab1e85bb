"""xb_ssm_conv and xb_ssm_scan against their formulas in 64 bits (tests/ssm_oracle.py, where the bounds come from)."""
import numpy as np
import pytest
import torch

import pkg
import ssm_oracle

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    pkg.load()
    from x_deeplearning_b200 import capi, ops
    return ops, capi


def _np(t):
    return t.detach().double().cpu().numpy()


def _lists(case, rng):
    """(first, last) of every list, the rows, whether by offsets"""
    if isinstance(case, tuple):                        # (lists, rows each)
        n, t = case
        return [(i * t, (i + 1) * t) for i in range(n)], n * t, None
    off = np.concatenate([[0], np.cumsum(case)])
    return [(int(off[i]), int(off[i + 1])) for i in range(len(case))], int(off[-1]), off.astype(np.int32)


def _wide(rng, rows, cols, dtype, pad, skew, std=1.0):
    """[rows, cols] in a wider matrix whose rows begin `skew` columns in; what lies around it is NaN"""
    t = torch.full((max(rows, 1), cols + pad + skew), float("nan"), dtype=dtype, device="cuda")
    v = t[:rows, skew:skew + cols]
    v.copy_(torch.from_numpy(rng.normal(0, std, (rows, cols))).to(dtype))
    return v


LISTS = [(1, 1), (5, 1), (3, 7), (2, 100), [0, 1, 0, 5, 17, 0, 64, 2, 33, 0], [131, 1, 0, 260], [3, 0]]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("lists", LISTS, ids=str)
@pytest.mark.parametrize("D,K,pad,skew", [(1, 2, 0, 0), (36, 4, 0, 0), (72, 4, 8, 0), (131, 3, 0, 1), (200, 8, 3, 0), (520, 5, 8, 8)])
def test_conv(dtype, lists, D, K, pad, skew):
    ops, capi = _ops()
    rng = np.random.default_rng(D + K)
    lists, rows, off = _lists(lists, rng)
    behind = 9 if off is not None else 0
    x = _wide(rng, rows + behind, D, T_[dtype], pad, skew)
    x[rows:] = float("nan")
    out = torch.full((rows + behind, D + pad + skew), 5.0, dtype=T_[dtype], device="cuda")[:, skew:skew + D]
    t = lambda *s, std=1.0: torch.from_numpy(rng.normal(0, std, s)).to("cuda", T_[dtype])
    w, b = t(D, K, std=K ** -0.5), t(D, std=0.3)
    n = len(lists)
    slots = torch.from_numpy(rng.permutation(n + 3)[:n].astype(np.int32)).cuda()
    state = t(n + 3, K - 1, D)
    kw = dict(offsets=torch.from_numpy(off).cuda()) if off is not None else dict(T=rows // n)
    before = _np(state)
    at = slots.cpu().numpy()
    for silu in (True, False):
        want, bound, after = ssm_oracle.conv(_np(x), _np(w), _np(b), lists, before[at], silu, dtype)
        kept = torch.full_like(state, 7.0)
        out.fill_(5.0)
        ops.ssm_conv(x, w, b, state_in=state, state_out=kept, slots=slots, silu=silu, out=out, **kw)
        ssm_oracle.close(_np(out)[:rows], want[:rows], bound[:rows], "y")
        assert (out[rows:] == 5.0).all()
        np.testing.assert_array_equal(_np(kept)[at], np.stack(after))
        rest = np.setdiff1d(np.arange(n + 3), at)
        assert (_np(kept)[rest] == 7.0).all()
        # in place
        moved = state.clone()
        y = ops.ssm_conv(x, w, b, state_in=moved, state_out=moved, slots=slots, silu=silu, **kw)
        assert torch.equal(y[:rows], out[:rows]) and torch.equal(moved[slots.long()], kept[slots.long()])
        np.testing.assert_array_equal(_np(moved)[rest], before[rest])
    # no states, no bias; states kept of lists that begin with zeros
    want, bound, after = ssm_oracle.conv(_np(x), _np(w), np.zeros(D), lists, np.zeros((n, K - 1, D)), True, dtype)
    kept = torch.full((n, K - 1, D), 7.0, dtype=T_[dtype], device="cuda")
    y = ops.ssm_conv(x, w, state_out=kept, **kw)
    ssm_oracle.close(_np(y)[:rows], want[:rows], bound[:rows], "y without states")
    np.testing.assert_array_equal(_np(kept), np.stack(after))


def _scan_inputs(rng, rows, behind, D, N, groups, dtype, pad, skew):
    s = dict(x=_wide(rng, rows + behind, D, T_[dtype], pad, skew), delta=_wide(rng, rows + behind, D, T_[dtype], pad, skew, 0.6),
             z=_wide(rng, rows + behind, D, T_[dtype], pad, skew), B=_wide(rng, rows + behind, groups * N, T_[dtype], pad, skew),
             C=_wide(rng, rows + behind, groups * N, T_[dtype], pad, skew))
    for t in s.values():
        t[rows:] = float("nan")
    f = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()
    step = np.exp(rng.uniform(np.log(1e-3), np.log(0.5), D))
    s.update(A=f(-np.exp(rng.uniform(np.log(0.05), np.log(16), (D, N)))), skip=f(rng.normal(1, 0.3, D)),
             bias=f(step + np.log(-np.expm1(-step))))
    return s


def _scan_want(s, lists, groups, h0, dtype, gate=True, skip=True, bias=True, softplus=True):
    rows, D = s["x"].shape
    N = s["A"].shape[1]
    n = {k: _np(v) for k, v in s.items()}
    zero = np.zeros(D)
    return ssm_oracle.scan(n["x"], n["delta"], n["A"], n["B"].reshape(rows, groups, N), n["C"].reshape(rows, groups, N),
                           n["skip"] if skip else zero, n["z"] if gate else None, n["bias"] if bias else zero, groups, softplus, lists, h0,
                           dtype)


def _check_scan(dtype, lists, D, N, groups, pad, skew, longest=True):
    ops, capi = _ops()
    rng = np.random.default_rng(D * 100 + N)
    lists, rows, off = _lists(lists, rng)
    n, behind = len(lists), 7 if off is not None else 0
    s = _scan_inputs(rng, rows, behind, D, N, groups, dtype, pad, skew)
    out = torch.full((rows + behind, D + pad + skew), 5.0, dtype=T_[dtype], device="cuda")[:, skew:skew + D]
    slots = torch.from_numpy(rng.permutation(n + 3)[:n].astype(np.int32)).cuda()
    at, rest = slots.cpu().numpy(), np.setdiff1d(np.arange(n + 3), slots.cpu().numpy())
    state = torch.from_numpy(rng.normal(0, 0.5, (n + 3, D, N)).astype(np.float32)).cuda()
    kw = dict(offsets=torch.from_numpy(off).cuda(), longest=max(b - a for a, b in lists) if longest else 0) if off is not None else dict(T=rows // n)
    want, bound, last, elast = _scan_want(s, lists, groups, _np(state)[at], dtype)
    kept = torch.full_like(state, 7.0)
    ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], delta_bias=s["bias"], groups=groups, h_in=state, h_out=kept,
                 slots=slots, out=out, **kw)
    ssm_oracle.close(_np(out)[:rows], want[:rows], bound[:rows], "y")
    ssm_oracle.close(_np(kept)[at], np.stack(last), np.stack(elast), "states")
    assert (out[rows:] == 5.0).all() and (_np(kept)[rest] == 7.0).all()
    moved = state.clone()                              # in place: the same bits
    y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], delta_bias=s["bias"], groups=groups, h_in=moved,
                     h_out=moved, slots=slots, **kw)
    assert torch.equal(y[:rows], out[:rows]) and torch.equal(moved[slots.long()], kept[slots.long()])
    assert torch.equal(moved[torch.from_numpy(rest).cuda()], state[torch.from_numpy(rest).cuda()])
    # nothing optional
    want, bound, last, elast = _scan_want(s, lists, groups, np.zeros((n, D, N)), dtype, gate=False, skip=False, bias=False)
    kept = torch.full((n, D, N), 7.0, device="cuda")
    y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], groups=groups, h_out=kept, **kw)
    ssm_oracle.close(_np(y)[:rows], want[:rows], bound[:rows], "y without options")
    ssm_oracle.close(_np(kept), np.stack(last), np.stack(elast), "states without options")


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("lists", LISTS, ids=str)
@pytest.mark.parametrize("D,N,groups,pad,skew", [(1, 1, 1, 0, 0), (36, 16, 1, 0, 0), (72, 16, 2, 8, 0), (131, 5, 1, 0, 1), (48, 64, 3, 0, 0),
                                                 (40, 33, 1, 3, 2), (264, 8, 1, 8, 8), (20, 3, 4, 0, 0)])
def test_scan(dtype, lists, D, N, groups, pad, skew):
    _check_scan(dtype, lists, D, N, groups, pad, skew)


@pytest.mark.parametrize("dtype,lists,D,N,groups", [
    ("f32", (1, 9000), 8, 16, 1), ("f32", (2, 3001), 40, 16, 1), ("bf16", [5000, 1, 0, 700, 3, 2500, 0], 72, 16, 1),
    ("f16", [1] * 300 + [2000] + [0, 7] * 40, 36, 8, 1), ("f32", [0, 0, 2049, 4096, 31], 18, 64, 2), ("f32", [4000], 130, 4, 1),
    ("f32", [int(n) for n in np.random.default_rng(8).integers(0, 41, 900)] + [301], 24, 16, 1),
    ("bf16", (40, 200), 136, 16, 1), ("f16", (700, 20), 72, 16, 1), ("f32", [900, 10] * 20, 33, 13, 1)], ids=lambda v: str(v)[:40])
@pytest.mark.parametrize("longest", [True, False])
def test_scan_of_long_and_many_lists(dtype, lists, D, N, groups, longest):
    _check_scan(dtype, lists, D, N, groups, 0, 0, longest)


@pytest.mark.parametrize("lists", [(2, 1), (2, 6), [6, 0, 3]], ids=str)
def test_scan_without_softplus_and_at_its_ends(lists):
    """Steps given as they are, zero ones among them; pre-activations where softplus is its argument or next to nothing."""
    ops, capi = _ops()
    rng = np.random.default_rng(3)
    lists, rows, off = _lists(lists, rng)
    s = _scan_inputs(rng, rows, 0, 24, 16, 1, "f32", 0, 0)
    kw = dict(offsets=torch.from_numpy(off).cuda()) if off is not None else dict(T=rows // len(lists))
    zero = np.zeros((len(lists), 24, 16))
    s["delta"].copy_(torch.rand_like(s["delta"]) * 0.3)
    s["delta"][:, ::5] = 0
    want, bound, _, _ = _scan_want(s, lists, 1, zero, "f32", bias=False, softplus=False)
    y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], softplus=False, **kw)
    ssm_oracle.close(_np(y), want, bound, "steps as they are")
    s["delta"][:, 0::4], s["delta"][:, 1::4], s["delta"][:, 2::4], s["delta"][:, 3::4] = 25.0, -25.0, 120.0, -110.0
    s["z"][:, ::3], s["z"][:, 1::3] = 95.0, -95.0
    want, bound, _, _ = _scan_want(s, lists, 1, zero, "f32", bias=False)
    y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], **kw)
    # exp of -95 and less is below what a quotient's fast form keeps: absolute 2^-100 there
    ssm_oracle.close(_np(y), want, bound + 2.0 ** -100, "ends of softplus and gate")


def test_slots_outside_and_lists_alone():
    """A slot outside the table begins with zeros and is not kept; a list's NaN and infinities stay its own."""
    ops, capi = _ops()
    rng = np.random.default_rng(4)
    lists, rows, off = _lists([5, 70, 0, 9, 300], rng)
    s = _scan_inputs(rng, rows, 0, 40, 16, 1, "f32", 0, 0)
    state = torch.from_numpy(rng.normal(0, 0.5, (3, 40, 16)).astype(np.float32)).cuda()
    slots = torch.tensor([2, -1, 0, 3, 1], dtype=torch.int32, device="cuda")
    h0 = np.stack([_np(state)[2], np.zeros((40, 16)), _np(state)[0], np.zeros((40, 16)), _np(state)[1]])
    want, bound, last, elast = _scan_want(s, lists, 1, h0, "f32")
    kept = torch.full_like(state, 7.0)
    off = torch.from_numpy(off).cuda()
    y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], delta_bias=s["bias"], offsets=off, h_in=state,
                     h_out=kept, slots=slots)
    ssm_oracle.close(_np(y), want, bound, "y")
    for i, slot in ((0, 2), (2, 0), (4, 1)):
        ssm_oracle.close(_np(kept)[slot], last[i], elast[i], "state %d" % i)
    s["x"][10:12], s["delta"][20:22] = float("nan"), float("inf")          # list 1
    again = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], delta_bias=s["bias"], offsets=off, h_in=state,
                         h_out=kept, slots=slots)
    others = [r for r in range(rows) if not 5 <= r < 75]
    assert torch.equal(again[others], y[others]) and torch.equal(again[5:10], y[5:10]) and again[10:75].isnan().all()
    w, b, x = torch.randn(40, 4, device="cuda"), torch.randn(40, device="cuda"), torch.randn(rows, 40, device="cuda")
    st = torch.randn(3, 3, 40, device="cuda")
    kept = torch.full_like(st, 7.0)
    y = ops.ssm_conv(x, w, b, offsets=off, state_in=st, state_out=kept, slots=slots)
    h0 = np.stack([_np(st)[2], np.zeros((3, 40)), _np(st)[0], np.zeros((3, 40)), _np(st)[1]])
    want, bound, after = ssm_oracle.conv(_np(x), _np(w), _np(b), lists, h0, True, "f32")
    ssm_oracle.close(_np(y), want, bound, "conv")
    for i, slot in ((0, 2), (2, 0), (4, 1)):
        np.testing.assert_array_equal(_np(kept)[slot], after[i])
    x[10:12] = float("inf")
    again = ops.ssm_conv(x, w, b, offsets=off)
    assert torch.equal(again[75:], y[75:]) or torch.isfinite(again[75:]).all()


@pytest.mark.parametrize("rows", [0, 1, 70])
def test_many_lists_without_rows(rows):
    """Thousands of empty lists ahead of, between and behind the others: their states go from one array to the other."""
    ops, capi = _ops()
    rng = np.random.default_rng(rows)
    lens = [0] * 3000 + ([rows // 2] + [0] * 5000 + [rows - rows // 2] + [0] * 700 if rows else [])
    lists, rows, off = _lists(lens, rng)
    n, off = len(lens), torch.from_numpy(off).cuda()
    x, w, b, st = torch.randn(rows, 20, device="cuda"), torch.randn(20, 4, device="cuda"), torch.randn(20, device="cuda"), torch.randn(n, 3, 20, device="cuda")
    want, bound, after = ssm_oracle.conv(_np(x), _np(w), _np(b), lists, _np(st), True, "f32")
    kept, moved = torch.full_like(st, 7.0), st.clone()
    ssm_oracle.close(_np(ops.ssm_conv(x, w, b, offsets=off, state_in=st, state_out=kept)), want, bound, "y")
    np.testing.assert_array_equal(_np(kept), np.stack(after))
    ops.ssm_conv(x, w, b, offsets=off, state_in=moved, state_out=moved)
    assert torch.equal(moved, kept)
    ops.ssm_conv(x, w, b, offsets=off, state_out=kept)
    assert (kept[torch.tensor(lens) == 0] == 0.0).all()
    s = _scan_inputs(rng, rows, 0, 20, 12, 1, "f32", 0, 0)
    h = torch.randn(n, 20, 12, device="cuda")
    want, bound, last, elast = _scan_want(s, lists, 1, _np(h), "f32")
    kept, moved = torch.full_like(h, 7.0), h.clone()
    call = lambda **k: ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], delta_bias=s["bias"], offsets=off, **k)
    ssm_oracle.close(_np(call(h_in=h, h_out=kept)), want, bound, "y")
    ssm_oracle.close(_np(kept), np.stack(last), np.stack(elast), "states")
    call(h_in=moved, h_out=moved)
    assert torch.equal(moved, kept)


def test_offsets_that_are_none():
    """Offsets that fall back or lie outside are cut to the rows: nothing outside is read or written."""
    ops, capi = _ops()
    x = torch.randn(20, 24, device="cuda")
    w = torch.randn(24, 4, device="cuda")
    s = _scan_inputs(np.random.default_rng(5), 20, 0, 24, 16, 1, "f32", 0, 0)
    off = torch.tensor([-5, 4, 2, 9, 400], dtype=torch.int32, device="cuda")       # lists [0, 4), none, [2, 9), [9, 20)
    y = ops.ssm_conv(x, w, offsets=off)
    assert torch.equal(y[9:], ops.ssm_conv(x[9:], w))
    y = ops.ssm_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], offsets=off)
    one = ops.ssm_scan(s["x"][9:], s["delta"][9:], s["A"], s["B"][9:], s["C"][9:])
    np.testing.assert_allclose(_np(y[9:]), _np(one), rtol=1e-5, atol=1e-6)


def test_tokens_one_by_one_are_the_list():
    """A list walked as a whole, in two parts, and row by row from kept states; convolution and scan in turn."""
    ops, capi = _ops()
    rng = np.random.default_rng(6)
    n, t, D, N = 5, 37, 72, 16
    s = _scan_inputs(rng, n * t, 0, D, N, 1, "f32", 0, 0)
    w, b = torch.randn(D, 4, device="cuda") / 2, torch.randn(D, device="cuda")

    def walk(parts):
        conv, h = torch.zeros(n, 3, D, device="cuda"), torch.zeros(n, D, N, device="cuda")
        out = torch.empty(n, t, D, device="cuda")
        a = 0
        for m in parts:
            cut = lambda v: v.reshape(n, t, -1)[:, a:a + m].reshape(n * m, -1)
            u = ops.ssm_conv(cut(s["x"]), w, b, T=m, state_in=conv, state_out=conv)
            y = ops.ssm_scan(u, cut(s["delta"]), s["A"], cut(s["B"]), cut(s["C"]), D=s["skip"], z=cut(s["z"]), delta_bias=s["bias"], T=m,
                             h_in=h, h_out=h)
            out[:, a:a + m] = y.view(n, m, D)
            a += m
        return out, conv, h
    whole = walk([t])
    for parts in ([1] * t, [20, 17], [1, 2, 30, 4]):
        got = walk(parts)
        assert torch.equal(got[1], whole[1])
        for g, v in ((got[0], whole[0]), (got[2], whole[2])):
            np.testing.assert_allclose(_np(g), _np(v), rtol=2e-5, atol=2e-5)


def test_refusals():
    ops, capi = _ops()
    s = _scan_inputs(np.random.default_rng(7), 12, 0, 24, 16, 1, "f32", 0, 0)
    names = ("x", "delta", "A", "B", "C")
    call = lambda **k: ops.ssm_scan(*[{**s, **k}[n] for n in names], **{n: v for n, v in k.items() if n not in names})
    call()
    h = torch.zeros(2, 24, 16, device="cuda")
    for bad in (dict(T=5), dict(T=6, h_in=h[:1]), dict(T=6, h_in=h.half()), dict(T=6, h_in=h, h_out=torch.zeros(3, 24, 16, device="cuda")),
                dict(delta=s["delta"].half()), dict(B=s["B"][:, :15]), dict(x=s["x"].cpu()), dict(A=s["A"].double()), dict(groups=5),
                dict(z=s["x"][:6]), dict(x=s["x"].t().contiguous().t()), dict(offsets=torch.zeros(3, dtype=torch.int64, device="cuda")),
                dict(T=6, h_in=h, slots=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(out=torch.zeros(12, 25, device="cuda"))):
        with pytest.raises(capi.XbError):
            call(**bad)
    with pytest.raises(capi.XbError):
        ops.ssm_conv(s["x"], torch.zeros(24, 9, device="cuda"))
    with pytest.raises(capi.XbError):
        ops.ssm_conv(s["x"], torch.zeros(24, 4, device="cuda"), state_in=torch.zeros(1, 4, 24, device="cuda"))
    # empty calls
    e = torch.zeros(0, 24, device="cuda")
    assert ops.ssm_conv(e, torch.zeros(24, 4, device="cuda")).shape == (0, 24)
    assert ops.ssm_scan(e, e, s["A"], torch.zeros(0, 16, device="cuda"), torch.zeros(0, 16, device="cuda")).shape == (0, 24)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    h.fill_(2.0)
    kept = torch.zeros_like(h)
    ops.ssm_scan(e, e, s["A"], torch.zeros(0, 16, device="cuda"), torch.zeros(0, 16, device="cuda"), offsets=off, h_in=h, h_out=kept)
    assert (kept == 2.0).all()
