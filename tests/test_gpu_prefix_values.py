"""xb_prefix_attention: infinities and NaN of several rows at once, scores that are all -infinity, and many small weights beside a large one."""
import numpy as np
import pytest
import torch

import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    pkg.load()
    from x_deeplearning_b200 import ops
    return ops


def _normal(*shape, dtype, seed, std=0.3):
    return torch.from_numpy(np.random.default_rng(seed).normal(0, std, shape)).to("cuda", T_[dtype])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lists,T,prefix", [(1, 300, 0), (1, 300, 70), (1, 40, 20_000), (1, 300, 3000), (2500, 40, 0), (2500, 40, 70)])
def test_two_bad_rows(dtype, d, lists, T, prefix):
    """A NaN among the keys of one row and an infinity among the values of another: whoever sees both has NaN. So has who sees infinities of both signs."""
    ops = _ops()
    q, k, v = (_normal(lists * T, 2, d, dtype=dtype, seed=s) for s in range(3))
    kw = dict(scale=d ** -0.5, T=T)
    if prefix:
        kw.update(prefix_k=_normal(prefix, 2, d, dtype=dtype, seed=3), prefix_v=_normal(prefix, 2, d, dtype=dtype, seed=4))
    good = ops.prefix_attention(q, k, v, **kw)
    first = lists // 2 * T
    a, b, end = first + 10, first + 25, first + T
    for nan, inf in ((a, b), (b, a)):
        bad_k, bad_v = k.clone(), v.clone()
        bad_k[nan, 0, 5], bad_v[inf, 0, 3] = float("nan"), float("inf")
        y = ops.prefix_attention(q, bad_k, bad_v, **kw)
        assert torch.equal(y[:a], good[:a]) and torch.equal(y[end:], good[end:]) and torch.equal(y[:, 1], good[:, 1])
        assert torch.isnan(y[nan:end, 0].float()).all()
        if inf < nan:
            assert (y[inf:nan, 0, 3] == float("inf")).all() and torch.equal(y[inf:nan, 0, 4:], good[inf:nan, 0, 4:])
    bad_v = v.clone()
    bad_v[a, 0, 3], bad_v[b, 0, 3] = float("inf"), float("-inf")
    y = ops.prefix_attention(q, k, bad_v, **kw)
    assert (y[a:b, 0, 3] == float("inf")).all() and torch.isnan(y[b:end, 0, 3].float()).all()
    assert torch.equal(y[:, 0, 4:], good[:, 0, 4:]) and torch.equal(y[:a], good[:a]) and torch.equal(y[end:], good[end:])
    if prefix:
        for at in (0, prefix - 1):
            bad_v, bad_pv = v.clone(), kw["prefix_v"].clone()
            bad_pv[at, 0, 3], bad_v[a, 0, 3] = float("inf"), float("-inf")
            y = ops.prefix_attention(q, k, bad_v, **{**kw, "prefix_v": bad_pv})
            assert torch.isnan(y[a:end, 0, 3].float()).all()
            assert (y[:a, 0, 3] == float("inf")).all() and (y[end:, 0, 3] == float("inf")).all()
            assert torch.equal(y[:, 0, 4:], good[:, 0, 4:]) and torch.equal(y[:, 1], good[:, 1])
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_that_are_all_minus_infinity(dtype, d):
    """Rows that see such keys alone are 0 / 0; with a finite score beside them these keys take no part; a row that sees no key has zeros."""
    ops = _ops()
    inf = float("inf")
    lens, own = [3, 1, 130, 2, 300], [3, 0, 130, 1, 300]
    off, own_off = (torch.tensor(np.r_[0, np.cumsum(n)], dtype=torch.int32, device="cuda") for n in (lens, own))
    starts, own_starts = np.r_[0, np.cumsum(lens)], np.r_[0, np.cumsum(own)]
    q, k, v = _normal(sum(lens), 2, d, dtype=dtype, seed=0), _normal(sum(own), 1, d, dtype=dtype, seed=1), _normal(sum(own), 1, d, dtype=dtype, seed=2)
    q[:, :, 0] = 1.0
    kw = dict(offsets=off, own_offsets=own_off, scale=0.25)
    k[:, :, 0] = -inf
    y = ops.prefix_attention(q, k, v, **kw)
    none = torch.zeros(len(q), dtype=torch.bool, device="cuda")
    none[int(starts[1])] = True                                          # a list without own rows
    none[int(starts[3])] = True                                          # two queries, one own row: the first sees none
    assert (y[none] == 0).all() and torch.isnan(y[~none].float()).all()
    # a finite key in the middle of the last list
    k[int(own_starts[4]) + 140, 0, 0] = 0.0
    y = ops.prefix_attention(q, k, v, **kw)
    at = int(starts[4]) + 140
    assert torch.isnan(y[int(starts[4]):at].float()).all()
    assert torch.equal(y[at:], v[int(own_starts[4]) + 140].expand(2, d)[None].expand(len(q) - at, 2, d))
    # prefixes, short and of many CTAs, with and without such a key
    for n in (70, 256, 30_000):
        for rows in (1, 50, 300):
            pk, pv = _normal(n, 1, d, dtype=dtype, seed=3), _normal(n, 1, d, dtype=dtype, seed=4)
            pk[:, :, 0] = -inf
            call = dict(T=1, prefix_k=pk, prefix_v=pv, scale=0.25)
            q1 = q[:rows]
            assert torch.isnan(ops.prefix_attention(q1, **call).float()).all()
            pk[n // 3, 0, 0] = 0.0
            assert torch.equal(ops.prefix_attention(q1, **call), pv[n // 3].expand(2, d)[None].expand(rows, 2, d))
            pk[n // 3, 0, 0] = -inf
            k1, v1 = k[:rows].clone(), v[:rows]
            k1[:, :, 0] = 0.0
            assert torch.equal(ops.prefix_attention(q1, k1, v1, **call), v1.expand(rows, 2, d))
    assert ops.device_status() == 0


def test_many_small_weights():
    """fp16, 200 prefixes of 20 000 keys: one key of each takes all but 2^-26 for every other, whose values are 1 and the first one's 0.
    A weight is known to half of fp16's smallest step, 2^-25, where the largest is 2^7 or more: to 2^-32 of that, and 20 000 of them to 2^-17.7."""
    ops = _ops()
    n, d = 20_000, 8
    q = torch.zeros(200, 1, d, device="cuda", dtype=torch.float16)
    q[:, :, 0] = 1.0
    pk = torch.zeros(200, n, 1, d, device="cuda", dtype=torch.float16)
    pk[:, :, :, 0] = -18.0
    pk[:, 0] = 0.0
    pv = torch.ones(200, n, 1, d, device="cuda", dtype=torch.float16)
    pv[:, 0] = 0.0
    y = ops.prefix_attention(q, T=1, prefix_k=pk.flatten(0, 1), prefix_v=pv.flatten(0, 1), prefix_offsets=torch.arange(201, device="cuda", dtype=torch.int32) * n)
    rest = (n - 1) * np.exp(-18.0)
    want = rest / (1 + rest)
    assert np.abs(y.double().cpu().numpy() - want).max() <= n * 2.0 ** -32 + want * (2.0 ** -11 + 2.0 ** -15) + 2.0 ** -25


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_bad_values_of_long_lists(dtype, d):
    """One infinity in lists of 60 000 rows, whole, costs what its block costs: the call takes at most three times as long, and the rows ahead of it keep their bits."""
    ops = _ops()
    n = 60_000
    q, k, v = (_normal(2 * n, 1, d, dtype=dtype, seed=s) for s in range(3))
    kw = dict(scale=d ** -0.5, T=n)

    def run():
        at = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ops.prefix_attention(q, k, v, **kw)
        at[0].record()
        y = ops.prefix_attention(q, k, v, **kw)
        at[1].record()
        torch.cuda.synchronize()
        return y, at[0].elapsed_time(at[1])

    good, ms = run()
    for at in (0, 31_000, n - 1, n, n + 40_100):
        kept = v[at].clone()
        v[at, 0, 3] = float("inf")
        y, bad_ms = run()
        v[at] = kept
        end = n if at < n else 2 * n
        assert (y[at:end, 0, 3] == float("inf")).all()
        assert torch.equal(y[:at], good[:at]) and torch.equal(y[end:], good[end:]) and torch.equal(y[:, :, 4:], good[:, :, 4:])
        assert bad_ms < 3 * ms, (bad_ms, ms)
    assert ops.device_status() == 0
