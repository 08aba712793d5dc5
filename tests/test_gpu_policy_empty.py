"""No rows at all: each result of gated_residual_norm still has a gradient for each operand, like any other's."""
import pytest
import torch

from test_gpu_policy_ops import BF16, F32, block_problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)], ids=["f32", "bf16", "f32+bf16", "bf16+f32"])
@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64), (0, 5, 7)], ids=str)
@pytest.mark.parametrize("gated", [True, False])
def test_empty_reaches_every_operand(shape, types, gated):
    from rl4mm_amd import policy_ops as ops

    args, _, _ = block_problem(1, 0, shape[-1], *types)
    leaves = [(t.view(shape) if i < 3 else t).detach().requires_grad_(True) for i, t in enumerate(args)]
    if not gated:
        leaves[2] = None
    results = ops.gated_residual_norm(*leaves)
    wanted = [t for t in leaves if t is not None]
    for result, dtype in zip(results, types):
        assert result.shape == shape and result.dtype == dtype
        grads = torch.autograd.grad(result.sum(), wanted, retain_graph=True)
        assert all(g.shape == t.shape and g.dtype == t.dtype and not g.any() for g, t in zip(grads, wanted))
    with torch.no_grad():
        assert not any(t.requires_grad for t in ops.gated_residual_norm(*leaves))
