"""Calls of ops.ssm_conv, ops.ssm_scan, ops.lora_gemm and their C functions that are refused before anything runs: scratch that is not
there, sizes that 32-bit counts do not hold, results over their own inputs. Host logic alone."""
import ctypes as C

import pytest
import torch

import pkg
from test_ssm_lora_binding import bound  # noqa: F401  (a fixture)


def test_scratch_whose_bytes_are_one(bound):  # noqa: F811
    """An expanded vector has many elements and one byte."""
    ops, capi, seen, need, _ = bound
    x, w = torch.zeros(12, 24, dtype=torch.float16), torch.zeros(1, dtype=torch.uint8).expand(4096)
    need[0] = 1000
    with pytest.raises(capi.XbError, match="workspace"):
        ops.ssm_scan(x, x, torch.zeros(24, 16), x[:, :16], x[:, :16], workspace=w)
    with pytest.raises(capi.XbError, match="workspace"):
        ops.lora_gemm(x, torch.zeros(16, 24, dtype=torch.float16), torch.zeros(3, 8, 24, dtype=torch.float16), torch.zeros(3, 16, 8, dtype=torch.float16),
                      torch.zeros(12, dtype=torch.int32), trans_b=True, workspace=w)
    assert not seen
    ops.ssm_scan(x, x, torch.zeros(24, 16), x[:, :16], x[:, :16], workspace=torch.zeros(4096, dtype=torch.uint8)[:1])
    assert seen[-1][1][1] == 1
