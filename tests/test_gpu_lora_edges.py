"""xb_lora_gemm where single lanes, tables and sizes differ from the ordinary: against its formula in 64 bits (tests/ssm_oracle.py)."""
import numpy as np
import pytest
import torch

import pkg
import ssm_oracle
from test_gpu_lora import T_, _case, _check, _np, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N", [(700, 304), (2100, 304), (9600, 72)])
@pytest.mark.parametrize("r", [17, 32, 100, 128])
def test_lanes_of_a_warp_with_adapters_of_their_own(M, N, r):
    """Rows of a warp that take nothing of an adapter's U beside rows that do, for every column block of a rank above 16: one row in 32, every
    other one, and all but one."""
    rng = np.random.default_rng(M + r)
    s = _case(rng, M, 72, N, 3, r, "bf16", True, 0, "none")
    rows = np.arange(M)
    for own in (rows % 32 == 5, rows % 2 == 1, rows % 32 != 9):
        s["adapter"] = torch.from_numpy(np.where(own, rows // 128 % 3, -1).astype(np.int32)).cuda()
        _check(s, "bf16", "bf16", True)
    assert _ops()[0].device_status() == 0


@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("M,K,N,trans,pad", [(20, 32, 24, True, 0), (600, 72, 304, False, 0), (700, 250, 131, True, 1), (9600, 72, 40, True, 0),
                                             (513, 33, 17, False, 0)])
def test_without_adapters(dtype, out, M, K, N, trans, pad):
    """No adapters, and adapters of rank 0: the projection and its bias."""
    for n, r in ((0, 8), (3, 0)):
        s = _case(np.random.default_rng(M), M, K, N, n, max(r, 1), dtype, trans, pad, "none" if n == 0 else "mixed")
        if r == 0:
            s["A"], s["B"] = s["A"].new_empty((n, 0, K)), s["B"].new_empty((n, N, 0))
        _check(s, dtype, out, trans)


@pytest.mark.parametrize("M,K,N,r", [(3, 2, 65535 * 128 + 1, 1), (65535 * 64 + 65, 2, 1, 3)])
@pytest.mark.parametrize("n", [0, 2])
def test_more_columns_or_rows_than_a_grid_of_16_bits(M, K, N, r, n):
    s = _case(np.random.default_rng(1), M, K, N, n, r, "f32", False, 0, "mixed" if n else "none")
    _check(s, "f32", "f32", False)


@pytest.mark.parametrize("M,N", [(60, 72), (2100, 304), (9600, 72)])
@pytest.mark.parametrize("r", [3, 16, 20, 64])
def test_infinities_of_an_adapter_are_the_formula_s(M, N, r):
    """An infinite weight of B gives its sign times U's in its column, for the rows of its adapter alone, whichever kernel makes it. (U, which the
    kernels round, is of one sign as long as it is not next to 0.)"""
    ops, capi = _ops()
    s = _case(np.random.default_rng(M + r), M, 64, N, 3, r, "bf16", True, 0, "mixed")
    call = lambda: ops.lora_gemm(s["X"], s["W"], s["A"], s["B"], s["adapter"], bias=s["bias"], scale=s["scale"], trans_b=True)
    y = call()
    s["B"][1, 5, r - 1], s["B"][1, 40, 0] = float("inf"), float("-inf")
    again = call()
    mine = s["adapter"] == 1
    u = s["X"].double() @ s["A"][1].double().T
    touched = torch.zeros_like(y, dtype=torch.bool)
    touched[mine, 5] = touched[mine, 40] = True
    assert torch.equal(again[~touched], y[~touched])
    for col, j, sign in ((5, r - 1, 1.0), (40, 0, -1.0)):
        sure = mine & (u[:, j].abs() > 1e-3)
        assert sure.sum() > 5 and torch.equal(again[sure, col].double(), sign * u[sure, j].sign() * float("inf"))
        assert not torch.isfinite(again[mine, col]).any()


@pytest.mark.parametrize("how", ["mixed", "runs", "one", "few", "none"])
@pytest.mark.parametrize("M,K,N,n,r,pad,trans", [(2100, 72, 304, 1000, 16, 0, True), (2100, 72, 304, 700, 40, 1, False), (520, 65, 304, 2000, 5, 1, True),
                                                 (9600, 72, 72, 40000, 8, 1, True), (2100, 520, 40, 2000, 100, 0, True)])
def test_tables_of_many_adapters(how, M, K, N, n, r, pad, trans):
    """Tables of which more than 32 MB would be laid out; rows that name all, some, one or none of their adapters."""
    s = _case(np.random.default_rng(n), M, K, N, n, r, "bf16", trans, pad, "mixed" if how == "few" else how)
    if how == "few":
        s["adapter"] = torch.from_numpy(np.random.default_rng(2).choice([n - 1, 7, n // 2, -1, n], M).astype(np.int32)).cuda()
    _check(s, "bf16", "bf16", trans)


@pytest.mark.parametrize("M,N,n", [(2100, 304, 4), (2100, 304, 2000), (9600, 72, 30000), (600, 131, 3000)])
@pytest.mark.parametrize("pad", [0, 1])
def test_adapters_that_share_their_matrices_in_two_steps(M, N, n, pad):
    """One A, one B, or both for all adapters, of which most have no row; each with its own scale."""
    for shared in ("A", "B", "AB"):
        s = _case(np.random.default_rng(M), M, 96, N, 4, 8, "bf16", True, pad, "none")
        for k in "AB":
            s[k] = s[k][:1].expand(n, -1, -1) if k in shared else s[k].repeat((n + 3) // 4, 1, 1)[:n]
        s["scale"] = torch.rand(n, device="cuda") + 0.5
        s["adapter"] = torch.from_numpy(np.random.default_rng(n).integers(-1, min(n, 300), M).astype(np.int32)).cuda()
        assert all(s[k].stride(0) == 0 for k in shared)
        _check(s, "bf16", "bf16", True)


def test_a_large_table_in_a_graph_whose_rows_name_others_at_each_replay():
    ops, capi = _ops()
    s = _case(np.random.default_rng(3), 2100, 72, 304, 1000, 16, "bf16", True, 1, "mixed")
    call = lambda: ops.lora_gemm(s["X"], s["W"], s["A"], s["B"], s["adapter"], bias=s["bias"], scale=s["scale"], trans_b=True)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = call()
    for seed, most in ((4, 1000), (5, 3), (6, 0), (7, 300)):
        s["adapter"].copy_(torch.from_numpy(np.random.default_rng(seed).integers(-1, most + 1, 2100) - (most == 0)).cuda())
        g.replay()
        assert torch.equal(y, call())


@pytest.mark.parametrize("dtype,trans", [("f16", True), ("bf16", False)])
@pytest.mark.parametrize("M,N", [(9, 1024), (400, 304), (960, 152), (2048, 24)])
def test_few_rows_at_every_split_of_the_depth(dtype, trans, M, N):
    """Depths next to where a part or its slices become one more, and parts of which the last have little or nothing."""
    for K in (248, 256, 264, 384, 392, 512, 520, 776, 1032, 1280, 1288, 1544, 2056, 3080, 6152):
        s = _case(np.random.default_rng(K), M, K, N, 3, 8, dtype, trans, 0, "mixed")
        _check(s, dtype, "f32", trans)


@pytest.mark.parametrize("dtype,out", [("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("M", [1, 63, 64, 65, 128, 129, 500])
@pytest.mark.parametrize("K,N,r,trans", [(250, 131, 12, False), (73, 600, 40, True), (31, 40, 4, False), (1, 3, 1, True)])
def test_few_rows_that_start_anywhere(dtype, out, M, K, N, r, trans):
    _check(_case(np.random.default_rng(M), M, K, N, 4, r, dtype, trans, 0, "mixed"), dtype, out, trans)
