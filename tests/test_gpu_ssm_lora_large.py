"""The state-space layer and the adapters on arrays of more than 2^31 elements, and from several threads at once: the last rows and states
against calls of their own."""
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


ROWS, D = (1 << 31) // 520 + 1000, 520                 # elements of x past 2^31


def test_convolution_and_scan():
    ops = _ops()
    x, w = _normal(ROWS, D), _normal(D, 4, seed=1)
    off = torch.tensor([0, 700, ROWS - 901, ROWS - 300, ROWS], dtype=torch.int32, device="cuda")
    y = ops.ssm_conv(x, w, offsets=off)
    for a, b in ((ROWS - 901, ROWS - 300), (ROWS - 300, ROWS)):
        assert torch.equal(y[a:b], ops.ssm_conv(x[a:b], w))
    del y
    delta, B = _normal(ROWS, D, seed=2), _normal(ROWS, 16, seed=3)
    A = -torch.rand(D, 16, device="cuda") - 0.5
    h = torch.zeros(4, D, 16, device="cuda")
    y = ops.ssm_scan(x, delta, A, B, B, offsets=off, h_out=h)
    for i, a, b in ((2, ROWS - 901, ROWS - 300), (3, ROWS - 300, ROWS)):
        last = torch.zeros(1, D, 16, device="cuda")
        alone = ops.ssm_scan(x[a:b], delta[a:b], A, B[a:b], B[a:b], h_out=last)
        # (other plans: sums of 16 terms and at most 601 rows in another order; results are rounded to bf16)
        torch.testing.assert_close(y[a:b].float(), alone.float(), rtol=2.0 ** -7, atol=1e-4)
        torch.testing.assert_close(h[i], last[0], rtol=1e-4, atol=1e-5)


def test_single_rows_whose_states_pass_32_bits():
    ops = _ops()
    n, D, N = (1 << 31) // (512 * 16) + 100, 512, 16
    x, B, A = _normal(n, D), _normal(n, N, seed=1), -torch.rand(D, N, device="cuda")
    w, st = _normal(D, 8, seed=2), _normal(n, 7, D, seed=3)
    h = torch.zeros(n, D, N, device="cuda")
    h[-5:].normal_()
    kept = h[-5:].clone()
    y = ops.ssm_scan(x, x, A, B, B, T=1, h_in=h, h_out=h)
    want = ops.ssm_scan(x[-5:], x[-5:], A, B[-5:], B[-5:], T=1, h_in=kept, h_out=kept)
    assert torch.equal(y[-5:], want) and torch.equal(h[-5:], kept)
    kept = st[-5:].clone()
    y = ops.ssm_conv(x, w, T=1, state_in=st, state_out=st)
    assert torch.equal(y[-5:], ops.ssm_conv(x[-5:], w, T=1, state_in=kept, state_out=kept)) and torch.equal(st[-5:], kept)


@pytest.mark.parametrize("K,N,dtype", [(D, 200, torch.bfloat16), (D, 520, torch.bfloat16), (D + 1, 24, torch.bfloat16), (D, 24, torch.float32)])
def test_adapters(K, N, dtype):
    """One step, two steps, rows laid out again, fp32; rows and results past 2^31 elements, where the last rows alone take another kernel."""
    ops = _ops()
    X, W = _normal(ROWS, K, dtype=dtype), _normal(N, K, dtype=dtype, seed=1) * K ** -0.5
    A, B = _normal(3, 8, K, dtype=dtype, seed=2) * K ** -0.5, _normal(3, N, 8, dtype=dtype, seed=3)
    ad = (torch.arange(ROWS, device="cuda") % 4).to(torch.int32)
    Y = ops.lora_gemm(X, W, A, B, ad, trans_b=True, out_dtype=torch.float32 if N == 24 else None)
    for a in (0, ROWS - 3000):
        want = X[a:a + 3000].double() @ W.double().T
        for i in range(3):
            m = ad[a:a + 3000] == i
            want[m] += X[a:a + 3000][m].double() @ A[i].double().T @ B[i].double().T
        # sums of at most 521 products of normal values in fp32, rounded once
        torch.testing.assert_close(Y[a:a + 3000].double(), want, rtol=2.0 ** -8 if Y.dtype == torch.bfloat16 else 1e-5, atol=2e-4)


def test_from_several_threads():
    """Calls of all kinds from four threads, each on a stream of its own: the same bits as alone."""
    ops = _ops()
    x, w = _normal(900, 72), _normal(72, 4, seed=1)
    A, B = -torch.rand(72, 16, device="cuda"), _normal(900, 16, seed=2)
    off = torch.tensor([0, 10, 400, 900], dtype=torch.int32, device="cuda")
    X = {m: _normal(m, 256, seed=m) for m in (40, 3000)}
    W, a, b = _normal(304, 256, seed=4), _normal(5, 8, 256, seed=5), _normal(5, 304, 8, seed=6)
    ad = {m: (torch.arange(m, device="cuda") % 6).to(torch.int32) for m in X}
    calls = [lambda: ops.ssm_conv(x, w, offsets=off), lambda: ops.ssm_scan(x, x, A, B, B, offsets=off)] + [
        lambda m=m: ops.lora_gemm(X[m], W, a, b, ad[m], trans_b=True) for m in X]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(30):
                    j = (i + k) % len(calls)
                    y = calls[j]()
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(y, want[j]):
                        bad.append(j)
        except Exception as e:                         # (shown by the assertion below)
            bad.append(repr(e))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
