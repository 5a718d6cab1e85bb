"""xb_lora_gemm against its formula in 64 bits (tests/ssm_oracle.py, where the bounds come from)."""
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


def _case(rng, M, K, N, n, r, dtype, trans, pad, how):
    dt = T_[dtype]

    def t(*shape, std=1.0):
        full = torch.full(shape[:-1] + (shape[-1] + pad,), float("nan"), dtype=dt, device="cuda")
        v = full[..., :shape[-1]]
        v.copy_(torch.from_numpy(rng.normal(0, std, shape)).to(dt))
        return v
    s = dict(X=t(M, K), W=t(N, K, std=K ** -0.5) if trans else t(K, N, std=K ** -0.5), A=t(n, r, K, std=K ** -0.5), B=t(n, N, r, std=r ** -0.5))
    s["scale"] = torch.from_numpy(rng.uniform(0.5, 2, n).astype(np.float32)).cuda()
    s["bias"] = torch.from_numpy(rng.normal(0, 0.3, N).astype(np.float32)).cuda()
    a = {"runs": np.sort(rng.integers(-1, n + 1, M)), "mixed": rng.integers(-1, n + 1, M), "one": np.full(M, n - 1), "none": np.full(M, -7)}[how]
    s["adapter"] = torch.from_numpy(a.astype(np.int32)).cuda()
    return s


def _check(s, dtype, out, trans, **more):
    ops, capi = _ops()
    M, N = s["X"].shape[0], s["W"].shape[0 if trans else 1]
    W = _np(s["W"])
    for with_scale, with_bias in ((True, True), (False, False)):
        want, bound = ssm_oracle.lora(_np(s["X"]), W.T if trans else W, _np(s["A"]), _np(s["B"]), s["adapter"].cpu().numpy(),
                                      _np(s["scale"]) if with_scale else np.ones(len(s["A"])), _np(s["bias"]) if with_bias else np.zeros(N), out)
        Y = torch.full((M + 2, N + 3), 5.0, dtype=T_[out], device="cuda")
        got = ops.lora_gemm(s["X"], s["W"], s["A"], s["B"], s["adapter"], bias=s["bias"] if with_bias else None,
                            scale=s["scale"] if with_scale else None, trans_b=trans, Y=Y[1:M + 1, 1:N + 1], **more)
        ssm_oracle.close(_np(got), want, bound, "with scale and bias" if with_scale else "without")
        Y[1:M + 1, 1:N + 1] = 5.0
        assert (Y == 5.0).all()                        # nothing beside the result was written
    return got


@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("how", ["runs", "mixed", "one", "none"])
@pytest.mark.parametrize("M,K,N,n,r,trans,pad", [
    (1, 16, 8, 1, 1, True, 0), (7, 40, 24, 3, 4, False, 0), (64, 72, 80, 64, 16, True, 8), (129, 250, 131, 5, 12, False, 0),
    (300, 324, 200, 4, 8, True, 4), (1000, 64, 256, 7, 16, True, 0), (513, 128, 48, 2, 64, False, 0), (260, 88, 176, 3, 32, True, 8),
    (130, 16, 8, 200, 3, True, 0), (256, 200, 80, 1, 100, True, 0), (700, 512, 304, 6, 24, True, 0), (600, 72, 40, 3, 100, False, 0),
    (1111, 324, 200, 12, 8, True, 4), (2000, 640, 520, 40, 16, True, 0), (513, 1280, 1024, 3, 128, True, 0), (900, 24, 1000, 5, 33, False, 0),
    (640, 136, 17, 9, 20, True, 0), (9600, 72, 200, 12, 8, True, 0), (10001, 136, 24, 40, 16, False, 0), (9473, 24, 190, 3, 64, True, 0),
    (12000, 200, 240, 2, 5, True, 0), (9999, 72, 81, 6, 30, True, 0), (20000, 16, 232, 1, 16, False, 0)])
def test_lora(dtype, out, how, M, K, N, n, r, trans, pad):
    rng = np.random.default_rng(M + K + N)
    _check(_case(rng, M, K, N, n, r, dtype, trans, pad, how), dtype, out, trans)


def test_more_rows_than_a_turn():
    """fp32 rows beyond one turn of the addend's workspace"""
    rng = np.random.default_rng(9)
    s = _case(rng, 9000, 24, 2048, 3, 2, "f32", True, 0, "mixed")
    _check(s, "f32", "f32", True)


@pytest.mark.parametrize("M", [200, 700])
def test_wide_range_of_the_intermediate(M):
    """U = X A^T far above what fp16 holds, and far below its normal numbers, with results that fit."""
    ops, capi = _ops()
    rng = np.random.default_rng(10)
    for up, down in ((2.0 ** 9, 2.0 ** -14), (2.0 ** -11, 2.0 ** 9)):
        s = _case(rng, M, 256, 64, 2, 8, "f16", True, 0, "runs")
        s["X"] = (s["X"] * (up if up > 1 else 0.1)).contiguous()
        s["A"] = (s["A"] * up).contiguous()
        s["B"] = (s["B"] * down).contiguous()
        s["W"] = (s["W"] * (2.0 ** -6)).contiguous()
        _check(s, "f16", "f16", True)


@pytest.mark.parametrize("M", [400, 1300])
def test_bad_values_stay_in_their_rows(M):
    """A row's NaN or infinity, and an adapter that no row names, reach no other row."""
    ops, capi = _ops()
    rng = np.random.default_rng(11)
    s = _case(rng, M, 128, 96, 4, 16, "f16", True, 0, "mixed")
    s["adapter"].clamp_(max=2)
    call = lambda: ops.lora_gemm(s["X"], s["W"], s["A"], s["B"], s["adapter"], bias=s["bias"], scale=s["scale"], trans_b=True)
    y = call()
    s["X"][17], s["X"][250], s["A"][3], s["B"][3] = float("nan"), float("inf"), float("nan"), float("inf")
    again = call()
    others = [m for m in range(M) if m not in (17, 250)]
    assert torch.equal(again[others], y[others]) and not torch.isfinite(again[17]).any() and not torch.isfinite(again[250]).all()


@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("M,K,N,n,r,trans", [
    (600, 1, 24, 3, 2, True), (520, 5, 40, 2, 3, False), (511, 3, 8, 2, 1, True), (600, 72, 304, 300, 12, True), (9500, 72, 200, 300, 8, True),
    (9500, 40, 304, 2, 128, False), (700, 2000, 1, 5, 40, True),
    (1, 64, 10000, 3, 8, True), (64, 72, 10000, 40, 16, False), (200, 136, 2800, 9, 64, True), (2048, 72, 136, 9, 24, True), (2049, 72, 136, 9, 24, False),
    (70, 648, 72, 5, 128, True), (300, 64, 104, 3, 104, False), (65, 64, 33, 3, 100, True)])
def test_shallow_products_and_tiles_of_many_adapters(dtype, out, M, K, N, n, r, trans):
    s = _case(np.random.default_rng(K + n), M, K, N, n, r, dtype, trans, 0, "mixed")
    _check(s, dtype, out, trans)


@pytest.mark.parametrize("M,N", [(60, 72), (700, 300), (9600, 72)])
def test_adapters_that_share_their_matrices(M, N):
    """One A or one B for all adapters (a stride of 0), each with its own scale."""
    for shared in ("A", "B"):
        s = _case(np.random.default_rng(M), M, 96, N, 4, 8, "bf16", True, 0, "mixed")
        s[shared] = s[shared][:1].expand(4, -1, -1)
        assert s[shared].stride(0) == 0
        _check(s, "bf16", "bf16", True)


@pytest.mark.parametrize("M", [60, 700, 9600])
def test_infinities_of_one_sign_are_infinities(M):
    ops, capi = _ops()
    for r in (3, 16, 20):
        s = _case(np.random.default_rng(M + r), M, 64, 72, 2, r, "bf16", True, 0, "one")
        W, A, B = s["W"].abs() + 0.01, s["A"].abs() + 0.01, s["B"].abs() + 0.01
        s["X"][M // 2, 5] = float("inf")
        y = ops.lora_gemm(s["X"], W, A, B, s["adapter"], trans_b=True)
        assert (y[M // 2] == float("inf")).all() and torch.isfinite(y[:M // 2]).all() and torch.isfinite(y[M // 2 + 1:]).all()


def test_the_same_bits_each_time_and_on_other_streams():
    ops, capi = _ops()
    rng = np.random.default_rng(12)
    s = _case(rng, 3000, 324, 200, 12, 8, "f16", True, 4, "runs")
    call = lambda: ops.lora_gemm(s["X"], s["W"], s["A"], s["B"], s["adapter"], bias=s["bias"], scale=s["scale"], trans_b=True)
    y = call()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(g, y) for g in got)


def test_refusals():
    ops, capi = _ops()
    s = _case(np.random.default_rng(13), 20, 32, 24, 3, 4, "f16", True, 0, "mixed")
    call = lambda **k: ops.lora_gemm(*[{**s, **k}[n] for n in ("X", "W", "A", "B", "adapter")], trans_b=True, **{n: v for n, v in k.items() if n not in ("X", "W", "A", "B", "adapter")})
    call()
    for bad in (dict(W=s["W"][:, :31]), dict(A=s["A"].float()), dict(B=s["B"][:2]), dict(adapter=s["adapter"].long()),
                dict(adapter=s["adapter"][:19]), dict(bias=s["bias"].half()), dict(scale=s["scale"][:2]), dict(out_dtype=torch.bfloat16),
                dict(X=s["X"].cpu()), dict(Y=torch.zeros(20, 23, dtype=torch.float16, device="cuda")),
                dict(A=torch.zeros(3, 129, 32, dtype=torch.float16, device="cuda"), B=torch.zeros(3, 24, 129, dtype=torch.float16, device="cuda")),
                dict(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(capi.XbError):
            call(**bad)
    e = ops.lora_gemm(s["X"][:0], s["W"], s["A"], s["B"], s["adapter"][:0], trans_b=True)
    assert e.shape == (0, 24)
    # no adapters at all: the projection alone
    y = ops.lora_gemm(s["X"], s["W"], s["A"][:0], s["B"][:0], s["adapter"], bias=s["bias"], scale=s["scale"][:0], trans_b=True)
    assert torch.isfinite(y).all()
