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
@pytest.mark.parametrize("widths, room, most", [((32, 32), 1024, 384), ((64, 48), 1024, 208), ((128, 128), 512, 160), ((20, 100), 512, 160)], ids=str)
def test_as_many_as_fit(widths, room, most, dtype):
    for steps in (512, 700, 1024, 4096, 18000, 1_000_000):
        for units in (1, 2, 7, 37, 75, 79, 80, 100, 103, 104, 150, 159, 160, 207, 208, 300, 383, 384, 4096):
            n = parts(steps, units, *widths, dtype)
            limit = most // 2 if steps < 1024 and widths != (32, 32) else most
            assert (n == 1) if units >= limit else (1 < n and n * units <= room), (steps, units, n)
            assert (n - 1) * 128 < steps
    for steps in (1, 64, 128, 511):
        assert parts(steps, 1, *widths, dtype) == 1
