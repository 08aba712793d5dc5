"""CPU-only: into how many parts decay attention splits its steps, told by the workspace that holds a state and a carry for each."""
import ctypes as C

import pytest

from rl4mm_amd import _lib, _policy_capi as capi


def parts(steps, units, dk, dv, dtype):
    a = capi.Attention(dtype=dtype, heads=1, dk=dk, dv=dv, steps=steps, envs=units, scale=1.0, log_decay=64)
    size = _lib.policy_binding().fn["attention_workspace"](C.byref(a))
    one = units * (dk * dv + 1) * 4
    assert size >= 0 and size % one == 0
    return max(1, size // one)


@pytest.mark.parametrize("dtype", [capi.F32, capi.BF16])
@pytest.mark.parametrize("widths, room", [((32, 32), 1024), ((64, 48), 1024), ((128, 128), 512), ((20, 100), 512)], ids=str)
def test_as_many_as_fit(widths, room, dtype):
    """no more workgroups than have room at once, no part shorter than 128 steps but the last, and no parts from some number of environments and heads on"""
    split = 0
    for steps in (512, 700, 1024, 4096, 18000, 1_000_000):
        counts = []
        for units in (1, 2, 7, 37, 75, 90, 100, 128, 150, 192, 220, 300, 383, 384, 4096):
            n = parts(steps, units, *widths, dtype)
            assert n == 1 or n * units <= room, (steps, units, n)
            assert (n - 1) * 128 < steps
            counts.append(n)
        assert counts == sorted(counts, reverse=True) and counts[4] > 1 and counts[-2:] == [1, 1]
        split, before = sum(n > 1 for n in counts), split
        assert split >= before  # (the more steps, the more units pay)
    for steps in (1, 64, 128, 511):
        assert parts(steps, 1, *widths, dtype) == 1
