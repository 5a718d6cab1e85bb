"""xb_prefix_attention against its formula in 64 bits (tests/heads_oracle.py, where the bounds come from)."""
import numpy as np
import pytest
import torch

import heads_oracle
import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    m = pkg.load()
    from x_deeplearning_b200 import capi, ops
    return ops, capi


def _np(t):
    return t.detach().double().cpu().numpy()


def _cuda(a):
    return torch.from_numpy(np.asarray(a, np.int32)).cuda()


def _pairs(off):
    return [(int(a), int(b)) for a, b in zip(off[:-1], off[1:])]


class Call:
    """Lists of `queries` rows with `own` own rows (None: the queries' own), prefix p of `prefixes` rows shared by the next members[p] lists after `ahead`"""

    def __init__(self, queries, own, prefixes, members, H, Hkv, d, dtype, ahead=0, behind=5, std=1.0, seed=0):
        rng = np.random.default_rng(seed + d + H)
        t = lambda *s: torch.from_numpy(rng.normal(0, std, s)).to("cuda", T_[dtype])
        self.dtype, self.d, self.scale = dtype, d, d ** -0.5
        self.off, self.own_off = np.concatenate([[0], np.cumsum(queries)]), np.concatenate([[0], np.cumsum(queries if own is None else own)])
        self.pre_off, self.mem = np.concatenate([[0], np.cumsum(prefixes)]), ahead + np.concatenate([[0], np.cumsum(members)])
        self.rows = int(self.off[-1])
        self.q = t(self.rows + behind, H, d)
        self.q[self.rows:] = float("nan")
        more = behind if own is None else 7
        self.k, self.v = t(int(self.own_off[-1]) + more, Hkv, d), t(int(self.own_off[-1]) + more, Hkv, d)
        self.pk, self.pv = t(int(self.pre_off[-1]) + 3, Hkv, d), t(int(self.pre_off[-1]) + 3, Hkv, d)
        for x, n in ((self.k, self.own_off[-1]), (self.v, self.own_off[-1]), (self.pk, self.pre_off[-1]), (self.pv, self.pre_off[-1])):
            x[int(n):] = float("nan")                  # what belongs to no list
        self.kw = dict(offsets=_cuda(self.off), prefix_k=self.pk, prefix_v=self.pv, prefix_offsets=_cuda(self.pre_off), members=_cuda(self.mem), scale=self.scale)
        if own is not None:
            self.kw["own_offsets"] = _cuda(self.own_off)
        self.prefix_of = [next((tuple(map(int, self.pre_off[p:p + 2])) for p in range(len(prefixes)) if self.mem[p] <= i < self.mem[p + 1]), None)
                          for i in range(len(queries))]

    def want(self):
        return heads_oracle.prefix(_np(self.q)[:self.rows], _np(self.k), _np(self.v), _pairs(self.off), _pairs(self.own_off), self.prefix_of, _np(self.pk),
                                   _np(self.pv), self.scale, self.dtype)

    def run(self, **k):
        ops, capi = _ops()
        out = torch.full(self.q.shape, 5.0, device="cuda", dtype=self.q.dtype)
        y = ops.prefix_attention(self.q, self.k, self.v, out=out, **{**self.kw, **k})
        assert y.data_ptr() == out.data_ptr() and ops.device_status() == 0
        assert (out[self.rows:] == 5.0).all()
        return out[:self.rows]

    def check(self):
        y = self.run()
        heads_oracle.close(_np(y), *self.want(), "y")
        assert torch.equal(self.run(), y)
        return y


HEADS = [(1, 1, 64), (4, 2, 64), (2, 2, 128), (6, 2, 40), (8, 1, 72), (5, 1, 8), (3, 3, 120)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,d", HEADS)
@pytest.mark.parametrize("queries,own,prefixes,members,ahead", [
    ([1], [1], [5], [1], 0),
    ([1] * 5, [1] * 5, [300], [5], 0),
    ([1] * 130, [1] * 130, [100, 129], [70, 60], 0),
    ([1] * 40, [17, 0, 33, 150, 1] * 8, [128, 0, 257], [20, 1, 19], 0),
    ([3, 0, 1, 40, 128, 7], None, [64, 31], [2, 3], 1),
    ([200, 1, 300], None, [10], [1], 1),
    ([5, 4, 6], [2, 4, 300], [0, 50], [1, 2], 0),
], ids=["one", "branches", "candidates", "ragged", "whole", "long", "fewer_own"])
def test_formula(dtype, H, Hkv, d, queries, own, prefixes, members, ahead):
    Call(queries, own, prefixes, members, H, Hkv, d, dtype, ahead).check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,prefix", [(1, 9000), (128, 9000), (129, 20_001), (700, 5000)])
def test_long_prefixes(dtype, d, n, prefix):
    """Items that many CTAs share, joined by the last kernel; sharper scores too, whose maximum grows often."""
    for std in (1.0, 2.5):
        c = Call([1] * n, [1] * n, [prefix], [n], 2, 1, d, dtype, std=std)
        y = c.run()
        rows = np.unique(np.r_[0, n // 2, n - 1])
        pick = lambda pairs: [pairs[i] for i in rows]
        own = pick(_pairs(c.own_off))
        want, bound = heads_oracle.prefix(_np(c.q)[rows], _np(c.k), _np(c.v), [(i, i + 1) for i in range(len(rows))], own, [(0, prefix)] * len(rows), _np(c.pk),
                                          _np(c.pv), c.scale, dtype)
        heads_oracle.close(_np(y)[rows], want, bound, "y")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_forms_of_a_call(dtype):
    """Equal lists, one prefix for all, members and prefixes of equal parts, no prefix, no own rows: what offsets would say."""
    ops, _ = _ops()
    c = Call([4] * 6, None, [50, 50], [3, 3], 4, 2, 64, dtype, behind=0)
    y = c.check()
    args = dict(scale=c.scale, prefix_k=c.pk[:100], prefix_v=c.pv[:100])
    assert torch.equal(ops.prefix_attention(c.q, c.k, c.v, T=4, prefix_offsets=_cuda([0, 50, 100]), **args), y)
    assert torch.equal(ops.prefix_attention(c.q, c.k, c.v, T=4, members=_cuda([0, 3, 6]), **args), y)
    one = Call([4] * 6, None, [100], [6], 4, 2, 64, dtype, behind=0)
    assert torch.equal(ops.prefix_attention(one.q, one.k, one.v, T=4, prefix_k=one.pk[:100], prefix_v=one.pv[:100], scale=one.scale), one.check())
    none = ops.prefix_attention(c.q, c.k, c.v, T=4, scale=c.scale)
    heads_oracle.close(_np(none), *heads_oracle.prefix(_np(c.q), _np(c.k), _np(c.v), _pairs(c.off), _pairs(c.off), [None] * 6, None, None, c.scale, dtype), "no prefix")
    alone = ops.prefix_attention(c.q, T=4, prefix_offsets=_cuda([0, 50, 100]), **args)
    heads_oracle.close(_np(alone), *heads_oracle.prefix(_np(c.q), None, None, _pairs(c.off), [(0, 0)] * 6, c.prefix_of, _np(c.pk), _np(c.pv), c.scale, dtype),
                       "no own rows")
    assert ops.prefix_attention(c.q[:0], c.k[:0], c.v[:0], T=1, scale=1.0).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_strides(dtype):
    """Slices of one projection, heads outside rows, results off 16 bytes."""
    ops, _ = _ops()
    rng = np.random.default_rng(7)
    t = lambda *s: torch.from_numpy(rng.normal(0, 1, s)).to("cuda", T_[dtype])
    qkv, kept = t(77, 4 + 2 + 2, 48), t(2, 2, 90, 48)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    pk, pv = kept[0].transpose(0, 1), kept[1].transpose(0, 1)
    want = heads_oracle.prefix(*(_np(x) for x in (q, k, v)), [(i * 7, i * 7 + 7) for i in range(11)], [(i * 7, i * 7 + 7) for i in range(11)], [(0, 90)] * 11, _np(pk),
                               _np(pv), 0.2, dtype)
    out = torch.full((77, 5, 49), 5.0, device="cuda", dtype=T_[dtype])
    for y in (ops.prefix_attention(q, k, v, T=7, prefix_k=pk, prefix_v=pv, scale=0.2),
              ops.prefix_attention(q, k, v, T=7, prefix_k=pk, prefix_v=pv, scale=0.2, out=out[:, 1:, 1:])):
        heads_oracle.close(_np(y), *want, "y")
    assert (out[:, 0] == 5.0).all() and (out[:, :, 0] == 5.0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("d", [64, 128])
def test_a_bad_row_reaches_those_that_see_it(dtype, bad, d):
    c = Call([1, 1, 30, 1, 300], [40, 1, 30, 200, 300], [200, 150], [3, 2], 2, 1, d, dtype)
    good = c.run()
    row = lambda i: slice(int(c.off[i]), int(c.off[i + 1]))
    seen = torch.zeros(c.rows, dtype=torch.bool, device="cuda")
    for own, of_list, at, first in ((True, 0, 39, 0), (True, 3, 0, 0), (True, 2, 11, 11), (True, 4, 150, 150), (False, None, 60, 0), (False, None, 349, 0)):
        seen[:] = False
        if own:
            seen[row(of_list)] = True
            seen[row(of_list)][:first] = False
            at += int(c.own_off[of_list])
        else:
            seen[:int(c.off[3])] = at < 200
            seen[int(c.off[3]):] = at >= 200
        for which in ("k", "v") if own else ("pk", "pv"):
            t = getattr(c, which)
            kept = t[at].clone()
            t[at, 0, 3] = bad
            y = c.run()
            t[at] = kept
            assert torch.equal(y[~seen], good[~seen])
            if which in ("v", "pv"):
                assert not torch.isfinite(y[seen][:, :, 3].float()).any()
                assert torch.equal(y[seen][:, :, 4:], good[seen][:, :, 4:]) and torch.equal(y[seen][:, :, :3], good[seen][:, :, :3])
            elif bad != bad:
                assert torch.isnan(y[seen].float()).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_large_scores(dtype):
    """Scores far apart and of either sign: one key takes all; scores all far below zero; the type's lowest value among the keys."""
    ops, _ = _ops()
    q = torch.zeros(3, 1, 64, device="cuda", dtype=T_[dtype])
    q[:, 0, 0] = torch.tensor([200.0, -200.0, 0.0])
    pk = torch.zeros(300, 1, 64, device="cuda", dtype=T_[dtype])
    pk[:, 0, 0] = torch.linspace(-200, 200, 300)
    pv = torch.arange(300, device="cuda").to(T_[dtype])[:, None, None].expand(300, 1, 64).contiguous()
    y = ops.prefix_attention(q, T=1, prefix_k=pk, prefix_v=pv)
    assert (y[0] == pv[299]).all() and (y[1] == pv[0]).all()
    assert (y[2].float() - 149.5).abs().max() <= 149.5 * (2.0 ** -8 + 2.0 ** -7)            # equal weights; values and the result rounded
    pk[:, 0, 0] = torch.finfo(T_[dtype]).min if dtype == "f16" else -1e30
    y = ops.prefix_attention(q[:1], T=1, prefix_k=pk, prefix_v=pv)
    assert torch.isfinite(y.float()).all() and (y.float() - 149.5).abs().max() <= 149.5 * (2.0 ** -8 + 2.0 ** -7)


def test_members_that_are_cut():
    """Members and offsets past what exists end with it."""
    c = Call([1] * 6, [1] * 6, [40, 30], [4, 2], 2, 2, 64, "bf16")
    y = c.check()
    members, pre = c.kw["members"].clone(), c.kw["prefix_offsets"].clone()
    members[-1] = 1 << 30
    c.kw["prefix_k"], c.kw["prefix_v"] = c.pk[:70], c.pv[:70]
    pre[-1] = 1 << 30
    assert torch.equal(c.run(members=members, prefix_offsets=pre), y)


def test_captured_and_on_several_streams():
    """Two captured calls with a workspace each, and eager ones on other streams, at once; a replay sees lengths that changed."""
    ops, capi = _ops()
    c = Call([1] * 200, [3] * 200, [3000, 40], [90, 110], 4, 2, 128, "bf16", behind=0)
    want = c.run()
    outs, graphs, streams = [torch.empty_like(want) for _ in range(4)], [], [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            ops.prefix_attention(c.q, c.k, c.v, out=outs[i], **c.kw)
        graphs.append(g)
    for turn in range(4):
        if turn == 2:
            c.kw["prefix_offsets"].copy_(_cuda([0, 500, 3040]))
            c.kw["members"].copy_(_cuda([0, 10, 200]))
            want = c.run()
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(4):
            with torch.cuda.stream(streams[i]):
                if i < 2:
                    graphs[i].replay()
                else:
                    ops.prefix_attention(c.q, c.k, c.v, out=outs[i], **c.kw)
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want)
    assert ops.device_status() == 0
