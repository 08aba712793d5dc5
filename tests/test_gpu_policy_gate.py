"""The gate's gradient where the gate is all but open or shut: sigmoid(u) sigmoid(-u) holds its digits, however small it is."""
import pytest
import torch

import policy_reference as ref
from test_gpu_policy_ops import BF16, F32, block_problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rl4mm_amd import policy_ops

    return policy_ops


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, BF16)], ids=["f32", "bf16", "f32+bf16"])
@pytest.mark.parametrize("width", [30, 64, 512, 750, 1024, 1500, 4096, 8192])
def test_saturated_gates(ops, width, types):
    """dgate = f res bn post s (1 - s), s = sigmoid(u).  All but s (1 - s) is off as in block_tolerance (10 c worse of its terms); the exponential's argument is
    rounded twice and its value twice more, which makes (1 + |u|) 2^-23 of it, and that enters s and 1 - s: 2 (1 + |u|) 2^-23 of the product, 2^-21 with the
    reciprocal and the products' own roundings.  Then the result's rounding."""
    args, dy, dz = block_problem(width, 5, width, *types)
    levels = torch.tensor([0.0, 3.0, 8.0, 12.0, 16.0, 20.0, 30.0, 45.0, 60.0, 80.0, -3.0, -8.0, -16.0, -20.0, -45.0, -80.0], device="cuda")
    args[2] = levels[torch.arange(5 * width, device="cuda") % 16].view(5, width).to(types[1])
    leaves = [t.detach().requires_grad_(True) for t in args]
    y, z = ops.gated_residual_norm(*leaves, eps=1e-6)
    (got,) = torch.autograd.grad([y, z], leaves[2], [dy, dz])
    x, b, u, post, res, pre = (t.detach().double().cpu() for t in args)
    s, other = torch.sigmoid(u), torch.sigmoid(-u)  # (in 64 bits 1 - s has no digits left at 40)
    rb = (b.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    bn = b * rb
    yy = x + res * s * post * bn
    ry = (yy.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    yn, g = yy * ry, dz.double().cpu() * pre
    f = dy.double().cpu() + ry * (g - yn * (g * yn).mean(-1, keepdim=True))
    want = f * res * bn * post * s * other
    rms = lambda t: t.square().mean(-1, keepdim=True).sqrt()  # noqa: E731
    Y = x.abs() + (res * s * post * bn).abs()
    worse, ny = 1 + rms(Y) * ry, Y * ry
    F = dy.double().cpu().abs() + ry * (g.abs() + ny * rms(ny) * rms(g))
    c = (width + 64) * 2.0**-24
    relative = 10 * c * worse + 2 * (1 + u.abs()) * 2.0**-23 + 2.0**-21
    tol = (F * res * bn * post).abs() * s * other * relative + ref.HALF[types[1]] * want.abs() + 1e-37
    ref.close(got, want, tol, "dgate")
