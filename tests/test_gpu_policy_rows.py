"""The block's backward pass over as many workgroups as there are rows for them: few rows, of widths whose rows take a wave or a workgroup, aligned and not."""
import ctypes as C

import pytest
import torch

from test_gpu_policy_ops import BF16, F32, block_problem, check_block


@pytest.mark.parametrize("rows, width, parts", [(1, 64, 1), (4, 512, 1), (5, 512, 2), (5000, 512, 512), (1, 513, 1), (300, 750, 300), (512, 1024, 512), (600, 1024, 512), (3, 8192, 3), (5000, 8192, 512)])
def test_workspace(rows, width, parts):
    """room for a workgroup to every row that one works on at a time, 512 at most"""
    from rl4mm_amd import _lib, _policy_capi as capi

    b = capi.Block(rows=rows, width=width, eps=1e-6, x=64, block=64, post=64, res=64, pre=64)
    assert _lib.policy_binding().fn["block_workspace"](C.byref(b)) == 2 * parts * width * 4


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, BF16)], ids=["f32", "bf16", "f32+bf16"])
@pytest.mark.parametrize("rows, width", [(3, 750), (129, 750), (513, 750), (700, 513), (130, 1024), (515, 520), (9, 500), (600, 1500)], ids=str)
def test_few_rows(rows, width, types):
    from rl4mm_amd import policy_ops as ops

    args, dy, dz = block_problem(rows, rows, width, *types)
    got = check_block(ops, args, dy, dz)
    assert all(torch.equal(a, b) for a, b in zip(got, check_block(ops, args, dy, dz)))
