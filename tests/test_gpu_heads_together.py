"""Rotation, linear attention and attention on shared prefixes as a model calls them: queries, keys and values are slices of one projection, histories
are walked once, new behaviours and candidates go on from what they left. Every step against its formula in 64 bits, of what the step before it gave."""
import numpy as np
import pytest
import torch

import heads_oracle
import pkg

pytestmark = pytest.mark.gpu

T_ = {"f16": torch.float16, "bf16": torch.bfloat16}
H, HKV, D, W = 4, 2, 64, 96                                # heads of queries, of keys; their width; the model's


def _ops():
    pkg.load()
    from x_deeplearning_b200 import ops
    return ops


def _np(t):
    return t.detach().double().cpu().numpy()


def _cuda(a, dtype=np.int32):
    return torch.from_numpy(np.asarray(a, dtype)).cuda()


class Layer:
    def __init__(self, dtype, seed=0):
        self.rng = np.random.default_rng(seed)
        self.dtype = dtype
        self.w = self.normal(W, (H + 2 * HKV) * D) * W ** -0.5
        self.freqs = torch.exp(torch.arange(D // 2, dtype=torch.float64) * (-np.log(10000.0) / (D // 2))).float().cuda()
        self.qw, self.kw = (torch.from_numpy(1 + 0.1 * self.rng.normal(size=D)).float().cuda() for _ in range(2))
        self.decay = torch.log1p(-torch.exp2(-4 - torch.arange(H, dtype=torch.float32))).cuda()

    def normal(self, *s):
        return torch.from_numpy(self.rng.normal(size=s)).to("cuda", T_[self.dtype])

    def project(self, x, positions):
        """Queries and keys with norms, turned in place, and values: slices of one projection"""
        ops = _ops()
        y = ops.gemm(x, self.w, out_dtype=T_[self.dtype]).view(-1, H + 2 * HKV, D)
        q, k, v = y[:, :H], y[:, H:H + HKV], y[:, H + HKV:]
        ops.qk_norm_rope(q, k, positions, self.freqs, q_weight=self.qw, k_weight=self.kw, out_q=q, out_k=k)
        return q, k, v

    def check_project(self, x, positions, q, k):
        raw = _ops().gemm(x, self.w, out_dtype=T_[self.dtype]).view(-1, H + 2 * HKV, D)
        for got, part, w in ((q, raw[:, :H], self.qw), (k, raw[:, H:H + HKV], self.kw)):
            want, bound = heads_oracle.rope(_np(part), positions.cpu().numpy(), _np(self.freqs), _np(w), 1e-6, True, False, self.dtype)
            heads_oracle.close(_np(got), want, bound, "rotated")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_histories_then_new_behaviours_then_candidates(dtype):
    ops, m = _ops(), Layer(dtype)
    lengths = np.array([70, 0, 1, 300, 129])
    off = np.concatenate([[0], np.cumsum(lengths)])
    lists = [(int(a), int(b)) for a, b in zip(off[:-1], off[1:])]
    rows, users = int(off[-1]), len(lengths)
    x, positions = m.normal(rows, W), _cuda(np.concatenate([np.arange(n) for n in lengths]))
    q, k, v = m.project(x, positions)
    m.check_project(x, positions, q, k)

    # histories: states left in slots that are not in the lists' order
    slots = _cuda([6, 0, 3, 5, 1])
    states = torch.full((7, H, D, D), 9.0, device="cuda")
    states[slots.long()] = 0.0
    y = ops.linear_attention(q, k, v, m.decay, scale=D ** -0.5, offsets=_cuda(off), longest=300, h_in=states, h_out=states, slots=slots)
    want, bound, last, blast = heads_oracle.linear(_np(q), _np(k), _np(v), _np(m.decay), D ** -0.5, lists, [np.zeros((H, D, D))] * users, dtype)
    heads_oracle.close(_np(y), want, bound, "y")
    for i, s in enumerate(slots.tolist()):
        heads_oracle.close(_np(states[s]), last[i], blast[i], "states")
    assert (states[2] == 9.0).all() and (states[4] == 9.0).all()

    # whole lists by softmax as well, the rows themselves their own keys: causal
    y = ops.prefix_attention(q, k, v, offsets=_cuda(off), scale=D ** -0.5)
    heads_oracle.close(_np(y), *heads_oracle.prefix(_np(q), _np(k), _np(v), lists, lists, [None] * users, None, None, D ** -0.5, dtype), "causal")

    # one new behaviour a user goes on from the states
    kept = states.clone()
    x1, p1 = m.normal(users, W), _cuda(lengths)
    q1, k1, v1 = m.project(x1, p1)
    m.check_project(x1, p1, q1, k1)
    y1 = ops.linear_attention(q1, k1, v1, m.decay, scale=D ** -0.5, T=1, h_in=states, h_out=states, slots=slots)
    want, bound, last, blast = heads_oracle.linear(_np(q1), _np(k1), _np(v1), _np(m.decay), D ** -0.5, [(i, i + 1) for i in range(users)],
                                                   [_np(kept[s]) for s in slots.tolist()], dtype)
    heads_oracle.close(_np(y1), want, bound, "new behaviours")
    for i, s in enumerate(slots.tolist()):
        heads_oracle.close(_np(states[s]), last[i], blast[i], "states")

    # candidates of every user against the history, read once for all of a user's, and themselves
    each = np.array([9, 3, 150, 0, 40])
    mem, n = np.concatenate([[0], np.cumsum(each)]), int(each.sum())
    xc, pc = m.normal(n, W), _cuda(np.repeat(lengths, each))
    qc, kc, vc = m.project(xc, pc)
    yc = ops.prefix_attention(qc, kc, vc, T=1, prefix_k=k, prefix_v=v, prefix_offsets=_cuda(off), members=_cuda(mem), scale=D ** -0.5)
    ones = [(i, i + 1) for i in range(n)]
    heads_oracle.close(_np(yc), *heads_oracle.prefix(_np(qc), _np(kc), _np(vc), ones, ones, [lists[u] for u in np.repeat(np.arange(users), each)], _np(k), _np(v),
                                                     D ** -0.5, dtype), "candidates")
    assert ops.device_status() == 0


def test_a_captured_step():
    """Projection, rotation, a step of the states and the attention on a cache that grows, in one graph: replays with other inputs give the eager bits."""
    ops, m = _ops(), Layer("bf16")
    users, most = 6, 400
    x, positions, slots = m.normal(users, W), _cuda(np.zeros(users)), _cuda([4, 2, 0, 5, 1, 3])
    states, cache_k, cache_v = torch.zeros(users, H, D, D, device="cuda"), m.normal(most, HKV, D), m.normal(most, HKV, D)
    prefix = _cuda([0, 0, 0])
    members = _cuda([0, 2, users])

    def step():
        q, k, v = m.project(x, positions)
        a = ops.linear_attention(q, k, v, m.decay, T=1, h_in=states, h_out=states, slots=slots)
        b = ops.prefix_attention(q, k, v, T=1, prefix_k=cache_k, prefix_v=cache_v, prefix_offsets=prefix, members=members, scale=D ** -0.5)
        return a, b
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    states.zero_()
    for turn in range(4):
        x.copy_(m.normal(users, W))
        positions.fill_(100 * turn)
        prefix.copy_(_cuda([0, 60 * turn, 133 * turn]))
        before = states.clone()
        g.replay()
        torch.cuda.synchronize()
        after, got = states.clone(), [t.clone() for t in out]
        states.copy_(before)
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(after, states)
    assert ops.device_status() == 0
