"""An infinite operand: the results that it reaches are infinities and not-numbers as the formula has them, however many steps there are."""
import math

import pytest
import torch

import policy_reference as ref
from test_gpu_policy_ops import BF16, F32, problem, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rl4mm_amd import policy_ops

    return policy_ops


def same_kind(got, want, tolerance, what):
    """not-numbers and infinities in the same places, everything else within its tolerance"""
    got = got.detach().double().cpu()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        wrong = (kind(got) != kind(want)).nonzero()
        assert not len(wrong), f"{what}: {kind.__name__} at {wrong[0].tolist()}: {got[tuple(wrong[0])].item()} instead of {want[tuple(wrong[0])].item()}, and at {len(wrong) - 1} others"
    there = torch.isfinite(want)
    ref.close(got[there], want[there], tolerance[there], what)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("log_decay", [-0.01, -3.0])
@pytest.mark.parametrize("steps", [200, 511, 512, 700, 1100])  # (from 512 on the steps are split)
@pytest.mark.parametrize("which", ["k", "v", "state"])
@pytest.mark.parametrize("resets", [False, True])
def test_infinite_operands(ops, which, steps, log_decay, resets, dtype):
    p, dout, dlast = problem(3, steps, 3, 1, 32, 48, dtype)
    p["log_decay"] = torch.tensor([log_decay], device="cuda")
    p["reset"] = torch.zeros(steps, 3, dtype=torch.bool, device="cuda")
    if resets:
        p["reset"][[5, steps // 2 + 40], [0, 1]] = True
    clean = {**p, which: p[which].clone()}
    if which == "state":
        p["state"][0, 0, 3, 4], p["state"][1, 0, :, 7] = -math.inf, math.inf
        clean["state"][0, 0, 3, 4], clean["state"][1, 0, :, 7] = 0.0, 0.0
    else:
        for n, t in ((0, 77), (1, steps // 2), (2, steps - 1)):
            p[which][t, n, 0, 9], clean[which][t, n, 0, 9] = math.inf if n != 1 else -math.inf, 0.0
    want, tol = ref.attention(**p), ref.attention_tolerance(**clean)
    got = run(ops, p)
    for key in ("out", "state"):
        same_kind(got[key], want[key], tol[key], key)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("steps", [200, 700])
def test_infinite_gradients(ops, steps, dtype):
    """dout holds one: what flows back in front of it"""
    p, dout, dlast = problem(4, steps, 2, 1, 32, 48, dtype)
    p["log_decay"] = torch.tensor([-0.01], device="cuda")
    tidy = dout.clone()
    dout[steps - 9, 0, 0, 11], tidy[steps - 9, 0, 0, 11] = math.inf, 0.0
    want, tol = ref.attention(**p, dout=dout, dlast=dlast), ref.attention_tolerance(**p, dout=tidy, dlast=dlast)
    got = run(ops, p, dout, dlast)
    for key in ("dq", "dk", "dv", "dstate"):
        same_kind(got[key], want[key], tol[key], key)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("steps", [1, 5, 20, 32, 40, 100, 150, 700])
@pytest.mark.parametrize("width", [32, 64, 128])
def test_results_beyond_the_type(ops, width, steps, dtype):
    """All operands 1 and a scale of 1e38: every result that has the scale once is more than 32 bits hold, and infinite; none is no number."""
    q, k, v = (torch.ones(steps, 2, 1, width, dtype=dtype, device="cuda", requires_grad=True) for _ in range(3))
    out, last = ops.decay_attention(q, k, v, torch.tensor([-0.01], device="cuda"), scale=1e38)
    assert torch.isposinf(out).all() and torch.isfinite(last).all()
    for g in torch.autograd.grad(out, (q, k, v), torch.ones_like(out)):
        assert torch.isposinf(g).all()
