"""Decay attention in bfloat16 is as exact as float32 arithmetic rounded once (tests/policy_bits.py)."""
import pytest
import torch

import policy_reference as ref
from policy_bits import attention_bits
from test_gpu_policy_ops import BF16, problem, run

pytestmark = pytest.mark.gpu

SIZES = [  # T, N, H, dk, dv
    (1, 3, 2, 64, 64), (15, 2, 3, 32, 32), (20, 3, 2, 64, 64), (31, 2, 1, 20, 50), (32, 2, 2, 50, 20), (33, 2, 1, 64, 64), (63, 2, 1, 64, 32), (64, 2, 2, 64, 64), (64, 2, 1, 32, 32),
    (64, 2, 1, 128, 128), (100, 2, 1, 128, 128), (130, 2, 2, 24, 128), (150, 2, 2, 64, 64), (200, 2, 1, 33, 127), (257, 2, 1, 128, 32), (333, 2, 1, 48, 80), (20, 2, 1, 128, 128), (17, 2, 1, 5, 3),
]  # fmt: skip


@pytest.fixture(scope="module")
def ops():
    from rl4mm_amd import policy_ops

    return policy_ops


def check(ops, p, dout, dlast):
    want, tol = attention_bits(**p, dout=dout, dlast=dlast)
    got = run(ops, p, dout, dlast)
    for key, w in want.items():
        ref.close(got[key], w, tol[key], key)


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_rounded_once(ops, size):
    for resets, ragged in ((0.0, False), (0.03, True)):
        p, dout, dlast = problem(size[0] + ragged, *size, BF16, resets, ragged)
        check(ops, p, dout, dlast)


@pytest.mark.parametrize("size", [(5000, 1, 2, 32, 32), (1100, 3, 1, 128, 64), (700, 2, 1, 64, 64), (1030, 1, 1, 30, 21)], ids=str)
def test_rounded_once_on_a_long_axis(ops, size):
    p, dout, dlast = problem(3, *size, BF16, 0.001)
    p["log_decay"] = torch.tensor([-1e-4, -0.02][: size[2]], device="cuda")
    check(ops, p, dout, dlast)


def test_steps_are_the_segment_to_the_last_bit_or_two(ops):
    """A token at a time and the segment at once: each rounded once, so they differ by a rounding at most."""
    p, _, _ = problem(22, 75, 6, 2, 64, 64, BF16, 0.03)
    want, tol = attention_bits(**p)
    state, outs = p["state"].clone(), []
    for t in range(75):
        outs.append(ops.decay_attention_step(p["q"][t], p["k"][t], p["v"][t], p["log_decay"], state, reset=p["reset"][t], scale=p["scale"]))
    ref.close(torch.stack(outs), want["out"], tol["out"], "steps")
    ref.close(run(ops, p)["out"], want["out"], tol["out"], "segment")
