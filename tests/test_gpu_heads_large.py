"""The rotation, linear attention and attention on shared prefixes on arrays of more than 2^31 elements, and from several threads at once: the last
rows and states against calls of their own."""
import threading

import pytest
import torch

import pkg

pytestmark = pytest.mark.gpu


def _ops():
    pkg.load()
    from x_deeplearning_b200 import ops
    return ops


def _normal(*shape, dtype=torch.bfloat16, seed=0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=torch.Generator(device="cuda").manual_seed(seed))


STEP = 1 << 20                                             # elements between rows of the far-apart arrays: 2100 rows pass 2^31


def _far(rows, heads, d, seed):
    x = torch.empty(rows, STEP, device="cuda", dtype=torch.bfloat16)
    v = x[:, 1024:1024 + heads * d].view(rows, heads, d)
    v.copy_(_normal(rows, heads, d, seed=seed))
    return v


def test_rows_far_apart():
    """Rows of all inputs and results 2^20 elements apart: the same bits as the packed ones."""
    ops = _ops()
    n = 2100
    q, k, v = _far(n, 2, 64, 0), _far(n, 1, 64, 1), _far(n, 1, 64, 2)
    near = [t.contiguous() for t in (q, k, v)]
    y = torch.zeros(n, STEP, device="cuda", dtype=torch.bfloat16)[:, :128].view(n, 2, 64)
    positions, freqs = torch.arange(n, device="cuda", dtype=torch.int32), torch.logspace(0, -3, 32, device="cuda")
    a = ops.qk_norm_rope(q, None, positions, freqs, out_q=y)[0]
    assert torch.equal(a, ops.qk_norm_rope(near[0], None, positions, freqs)[0])
    decay = torch.tensor([-0.01, -0.2], device="cuda")
    off = torch.tensor([0, 700, n - 90, n], dtype=torch.int32, device="cuda")
    for of in (off, off[[0, 3]]):
        kw = dict(offsets=of, longest=n)
        assert torch.equal(ops.linear_attention(q, k, v, decay, out=y, **kw), ops.linear_attention(*near, decay, **kw))
    kw = dict(offsets=off, scale=0.125)
    assert torch.equal(ops.prefix_attention(q, k, v, out=y, **kw), ops.prefix_attention(*near, **kw))
    assert torch.equal(ops.prefix_attention(q, T=1, prefix_k=k, prefix_v=v, scale=0.125, out=y), ops.prefix_attention(near[0], T=1, prefix_k=near[1], prefix_v=near[2], scale=0.125))
    assert ops.device_status() == 0


def test_states_that_pass_32_bits():
    ops = _ops()
    n, H = (1 << 31) // (8 * 64 * 64) + 40, 8
    x, v, decay = _normal(n, H, 64), _normal(n, H, 64, seed=1), torch.full((H,), -0.1, device="cuda")
    h = torch.zeros(n, H, 64, 64, device="cuda")
    h[-5:].normal_()
    kept = h[-5:].clone()
    y = ops.linear_attention(x, x, v, decay, T=1, h_in=h, h_out=h)
    want = ops.linear_attention(x[-5:], x[-5:], v[-5:], decay, T=1, h_in=kept, h_out=kept)
    assert torch.equal(y[-5:], want) and torch.equal(h[-5:], kept)
    # lists of a few rows, their states in the last slots
    slots = torch.arange(n - 3, n, device="cuda", dtype=torch.int32)
    y = ops.linear_attention(x[:300], x[:300], v[:300], decay, T=100, h_in=h, h_out=h, slots=slots)
    kept = kept[2:].clone()
    want = ops.linear_attention(x[:300], x[:300], v[:300], decay, T=100, h_in=kept, h_out=kept)
    assert torch.equal(y, want) and torch.equal(h[-3:], kept)


def test_a_prefix_of_more_than_2_31_elements():
    """A cache whose last rows lie past 2^31 elements: a prefix there, as a prefix of an array of its own."""
    ops = _ops()
    rows = (1 << 31) // (8 * 128) + 5000
    k = torch.zeros(rows, 8, 128, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros(rows, 8, 128, device="cuda", dtype=torch.bfloat16)
    for t, seed in ((k, 0), (v, 1)):
        t[-4000:] = _normal(4000, 8, 128, seed=seed)
    q, off = _normal(200, 16, 128, seed=2), torch.tensor([0, 40, rows - 3999, rows], dtype=torch.int32, device="cuda")
    members = torch.tensor([0, 1, 1, 200], dtype=torch.int32, device="cuda")
    # (the plan of the whole call and of the part may differ: what is cut where, and so the order of sums of at most 3999 weights; results are rounded to bf16)
    y = ops.prefix_attention(q, T=1, prefix_k=k, prefix_v=v, prefix_offsets=off, members=members, scale=0.088)
    last = torch.tensor([0, 3999], dtype=torch.int32, device="cuda")
    want = ops.prefix_attention(q[1:], T=1, prefix_k=k[-3999:], prefix_v=v[-3999:], prefix_offsets=last, scale=0.088)
    torch.testing.assert_close(y[1:].float(), want.float(), rtol=2.0 ** -7, atol=1e-3)
    assert ops.device_status() == 0


def test_from_several_threads():
    """Calls of all kinds from four threads, each on a stream of its own: the same bits as alone."""
    ops = _ops()
    q, k, v = _normal(900, 4, 64), _normal(900, 2, 64, seed=1), _normal(900, 2, 64, seed=2)
    positions, freqs = torch.arange(900, device="cuda", dtype=torch.int32), torch.logspace(0, -3, 32, device="cuda")
    decay, off = torch.full((4,), -0.05, device="cuda"), torch.tensor([0, 10, 400, 900], dtype=torch.int32, device="cuda")
    h = torch.ones(900, 4, 64, 64, device="cuda")
    calls = [lambda: ops.qk_norm_rope(q, k, positions, freqs)[1], lambda: ops.linear_attention(q, k, v, decay, offsets=off),
             lambda: ops.linear_attention(q, k, v, decay, T=1, h_in=h), lambda: ops.linear_attention(q.float(), k.float(), v.float(), decay, offsets=off),
             lambda: ops.prefix_attention(q, k, v, offsets=off, scale=0.125), lambda: ops.prefix_attention(q, k, v, T=1, prefix_k=k, prefix_v=v, scale=0.125)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for n in range(30):
                    j = (n + i) % len(calls)
                    y = calls[j]()
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(y, want[j]):
                        bad.append(j)
        except Exception as e:                             # noqa: BLE001
            bad.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert bad == [] and ops.device_status() == 0
