"""xb_linear_attention against its recurrence in 64 bits (tests/heads_oracle.py, where the bounds come from)."""
import numpy as np
import pytest
import torch

import heads_oracle
import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    pkg.load()
    from x_deeplearning_b200 import capi, ops
    return ops, capi


def _np(t):
    return t.detach().double().cpu().numpy()


def _lists(case):
    """(first, last) of every list, the rows, offsets or none"""
    if isinstance(case, tuple):                        # (lists, rows each)
        n, t = case
        return [(i * t, (i + 1) * t) for i in range(n)], n * t, None
    off = np.concatenate([[0], np.cumsum(case)])
    return [(int(off[i]), int(off[i + 1])) for i in range(len(case))], int(off[-1]), off.astype(np.int32)


def _inputs(rng, rows, H, Hkv, dk, dv, dtype, std=1.0):
    t = lambda *s: torch.from_numpy(rng.normal(0, std, s)).to("cuda", T_[dtype])
    return t(rows, H, dk), t(rows, Hkv, dk), t(rows, Hkv, dv)


def _decays(H, fast=False):
    """Of a head that keeps all, slow ones, fast ones, and one without memory where there are many"""
    ld = np.log1p(-np.exp2(-4 - 6 * np.arange(H) / max(H - 1, 1)))
    if H > 1:
        ld[0] = 0.0
    if H > 2:
        ld[1] = -3.0
    if H > 3:
        ld[2] = -np.inf
    return torch.from_numpy(ld.astype(np.float32)).cuda()


LISTS = [(1, 1), (5, 1), (3, 7), (2, 100), (1, 64), [0, 1, 0, 5, 17, 0, 64, 2, 129, 0], [331, 1, 0, 460], [3, 0], (1, 1300)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("lists", LISTS, ids=str)
@pytest.mark.parametrize("H,Hkv,dk,dv", [(1, 1, 1, 1), (2, 2, 36, 36), (4, 2, 64, 64), (2, 1, 128, 128), (3, 3, 33, 70), (2, 2, 100, 24), (1, 1, 16, 127)])
def test_formula(dtype, lists, H, Hkv, dk, dv):
    ops, _ = _ops()
    rng = np.random.default_rng(dk + dv)
    lists, rows, off = _lists(lists)
    n, behind = len(lists), 9 if off is not None else 0
    q, k, v = _inputs(rng, rows + behind, H, Hkv, dk, dv, dtype)
    for t in (q, k, v):
        t[rows:] = float("nan")                        # rows behind the last list
    ld, scale = _decays(H), dk ** -0.5
    kw = dict(offsets=torch.from_numpy(off).cuda()) if off is not None else dict(T=rows // n)
    slots = torch.from_numpy(rng.permutation(n + 3)[:n].astype(np.int32)).cuda()
    at = slots.cpu().numpy()
    h = torch.from_numpy(rng.normal(0, 1, (n + 3, H, dk, dv)).astype(np.float32)).cuda()
    want, bound, last, elast = heads_oracle.linear(_np(q), _np(k), _np(v), _np(ld), scale, lists, _np(h)[at], dtype)
    out, kept = torch.full((rows + behind, H, dv), 5.0, dtype=T_[dtype], device="cuda"), torch.full_like(h, 7.0)
    ops.linear_attention(q, k, v, ld, scale=scale, h_in=h, h_out=kept, slots=slots, out=out, **kw)
    heads_oracle.close(_np(out)[:rows], want[:rows], bound[:rows], "y")
    assert (out[rows:] == 5.0).all()
    heads_oracle.close(_np(kept)[at], np.stack(last), np.stack(elast), "states")
    rest = np.setdiff1d(np.arange(n + 3), at)
    assert (kept[rest] == 7.0).all()
    # states moved on in place; the plan may go by the longest list
    moved = h.clone()
    y = ops.linear_attention(q, k, v, ld, scale=scale, h_in=moved, h_out=moved, slots=slots, **kw)
    assert torch.equal(y[:rows], out[:rows]) and torch.equal(moved[slots.long()], kept[slots.long()]) and torch.equal(moved[rest], h[rest])
    y = ops.linear_attention(q, k, v, ld, scale=scale, h_in=h, h_out=moved, slots=slots, longest=max(b - a for a, b in lists), **kw)
    heads_oracle.close(_np(y)[:rows], want[:rows], bound[:rows], "y, longest list known")
    # no states
    want, bound, last, elast = heads_oracle.linear(_np(q), _np(k), _np(v), _np(ld), scale, lists, np.zeros((n, H, dk, dv)), dtype)
    kept = torch.full((n, H, dk, dv), 7.0, device="cuda")
    y = ops.linear_attention(q, k, v, ld, scale=scale, h_out=kept, **kw)
    heads_oracle.close(_np(y)[:rows], want[:rows], bound[:rows], "y from zeros")
    heads_oracle.close(_np(kept), np.stack(last), np.stack(elast), "states from zeros")
    assert torch.equal(ops.linear_attention(q, k, v, ld, scale=scale, **kw)[:rows], y[:rows])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_strides_and_slots_outside(dtype):
    """Slices of one projection, rows off 16 bytes, heads outside rows; slots outside begin with zeros and are not kept; offsets cut to the rows."""
    ops, _ = _ops()
    rng = np.random.default_rng(3)
    H, dk, dv, lens = 3, 40, 48, [70, 5, 0, 129]
    lists, rows, off = _lists(lens)
    off_t = torch.from_numpy(off).cuda()
    ld = _decays(H)
    slots = torch.tensor([1, -1, 9, 0], dtype=torch.int32, device="cuda")
    h = torch.from_numpy(rng.normal(0, 1, (2, H, dk, dv)).astype(np.float32)).cuda()
    h0 = [_np(h)[1], np.zeros((H, dk, dv)), np.zeros((H, dk, dv)), _np(h)[0]]
    wide = torch.from_numpy(rng.normal(0, 1, (rows, H * (2 * dk + dv) + 8))).to("cuda", T_[dtype])
    for skew in (0, 1, 8):
        one = wide[:, skew:skew + H * (2 * dk + dv)]
        q, k, v = (t.unflatten(1, (H, -1)) for t in one.split([H * dk, H * dk, H * dv], 1))
        want, bound, last, elast = heads_oracle.linear(_np(q), _np(k), _np(v), _np(ld), 0.5, lists, h0, dtype)
        out = torch.full((H, rows, dv + 3), 5.0, device="cuda", dtype=T_[dtype])
        kept = torch.full_like(h, 7.0)
        ops.linear_attention(q, k, v, ld, scale=0.5, offsets=off_t, h_in=h, h_out=kept, slots=slots, out=out.transpose(0, 1)[:, :, :dv])
        heads_oracle.close(_np(out.transpose(0, 1)[:, :, :dv]), want, bound, "y")
        assert (out[:, :, dv:] == 5.0).all()
        heads_oracle.close(_np(kept)[[1, 0]], np.stack(last)[[0, 3]], np.stack(elast)[[0, 3]], "states")
    over = off_t.clone()
    over[-1] = rows + 1000                              # the last list ends with the rows
    y = ops.linear_attention(q, k, v, ld, scale=0.5, offsets=over, h_in=h, slots=slots)
    heads_oracle.close(_np(y), want, bound, "y")


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_row_stays_in_its_list(dtype, bad):
    """... and ahead of it: nothing of a row reaches an earlier one."""
    ops, _ = _ops()
    rng = np.random.default_rng(4)
    lists, rows, off = _lists([100, 90, 300, 65])
    q, k, v = _inputs(rng, rows, 2, 2, 64, 64, dtype)
    ld, kw = _decays(2), dict(offsets=torch.from_numpy(off).cuda())
    good = ops.linear_attention(q, k, v, ld, **kw)
    for t in (k, v):
        spoilt = t.clone()
        spoilt[130, 0, 5] = bad
        y = ops.linear_attention(q, spoilt if t is k else k, spoilt if t is v else v, ld, **kw)
        assert torch.equal(y[:130], good[:130]) and torch.equal(y[190:], good[190:]) and torch.equal(y[:, 1], good[:, 1])
        assert not torch.isfinite(y[130:190, 0]).all()


def test_small_and_large_values():
    """Values near the types' ends: sums stay fp32 whatever the inputs' type holds."""
    ops, _ = _ops()
    rng = np.random.default_rng(6)
    for dtype, std in (("f16", 3e-4), ("f16", 250.0), ("bf16", 1e-10), ("bf16", 1e8)):
        lists, rows, _ = _lists((2, 200))
        q, k, v = _inputs(rng, rows, 2, 2, 64, 64, dtype, std=std)
        q = (q.float() / std).to(T_[dtype])
        ld = _decays(2)
        scale = min(1.0, 1 / std)
        want, bound, last, elast = heads_oracle.linear(_np(q), _np(k), _np(v), _np(ld), scale, lists, np.zeros((2, 2, 64, 64)), dtype)
        kept = torch.empty(2, 2, 64, 64, device="cuda")
        y = ops.linear_attention(q, k, v, ld, scale=scale, T=200, h_out=kept)
        ok = np.abs(want) < (60000 if dtype == "f16" else 1e38)
        assert ok.mean() > 0.5
        heads_oracle.close(_np(y)[ok], want[ok], bound[ok], "y")
        heads_oracle.close(_np(kept), np.stack(last), np.stack(elast), "states")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_single_tokens_continue_a_list(dtype):
    """A list at once, and its first rows followed by one row a call on kept states."""
    ops, _ = _ops()
    rng = np.random.default_rng(8)
    H, dk, dv, T, n = 4, 64, 64, 90, 3
    q, k, v = (t.view(n, T, H, -1) for t in _inputs(rng, n * T, H, H, dk, dv, dtype))
    ld = _decays(H)
    want, bound, last, elast = heads_oracle.linear(*(_np(t.flatten(0, 1)) for t in (q, k, v)), _np(ld), 1.0, [(i * T, (i + 1) * T) for i in range(n)],
                                                   np.zeros((n, H, dk, dv)), dtype)
    h = torch.zeros(n, H, dk, dv, device="cuda")
    y = torch.empty(n, T, H, dv, device="cuda", dtype=T_[dtype])
    y[:, :70] = ops.linear_attention(*(t[:, :70].reshape(n * 70, H, -1) for t in (q, k, v)), ld, T=70, h_in=h, h_out=h).view(n, 70, H, dv)
    for t in range(70, T):
        y[:, t] = ops.linear_attention(q[:, t], k[:, t], v[:, t], ld, T=1, h_in=h, h_out=h)
    heads_oracle.close(_np(y.flatten(0, 1)), want, bound, "y")
    heads_oracle.close(_np(h), np.stack(last), np.stack(elast), "states")


def test_captured_and_on_several_streams():
    """Two captured calls with a workspace each, and eager ones on other streams, at once."""
    ops, _ = _ops()
    rng = np.random.default_rng(9)
    q, k, v = _inputs(rng, 6000, 2, 2, 64, 64, "bf16")
    ld = _decays(2)
    want = ops.linear_attention(q, k, v, ld, T=3000)
    outs, graphs, streams = [torch.empty_like(want) for _ in range(4)], [], [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            ops.linear_attention(q, k, v, ld, T=3000, out=outs[i])
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(4):
            with torch.cuda.stream(streams[i]):
                if i < 2:
                    graphs[i].replay()
                else:
                    ops.linear_attention(q, k, v, ld, T=3000, out=outs[i])
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want)
