"""Operands of one element to a row that torch negates on the way: the imaginary part of a conjugate."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def negated(*shape):
    z = torch.randn(*shape, dtype=torch.complex64, generator=torch.Generator().manual_seed(1)).cuda()
    t = torch.imag(z.conj())
    assert t.is_neg()
    return t, -torch.imag(z)


def test_negated_views():
    from rl4mm_amd import policy_ops as ops

    for width in (1, 3):
        lazy, plain = negated(5, 2, 2, width)
        decay = torch.tensor([-0.1, -0.2], device="cuda")
        ones = torch.ones(5, 2, 2, width, device="cuda")
        for q, k, v, want in ((lazy, ones, ones, (plain, ones, ones)), (ones, lazy, ones, (ones, plain, ones)), (ones, ones, lazy, (ones, ones, plain))):
            got, expected = ops.decay_attention(q, k, v, decay), ops.decay_attention(*want, decay)
            assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])
            one, two = torch.zeros(2, 2, width, width, device="cuda"), torch.zeros(2, 2, width, width, device="cuda")
            assert torch.equal(ops.decay_attention_step(q[0], k[0], v[0], decay, one), ops.decay_attention_step(*(t[0] for t in want), decay, two)) and torch.equal(one, two)
        leaf = torch.ones(5, 2, 2, width, device="cuda", requires_grad=True)
        grads = [torch.autograd.grad(ops.decay_attention(leaf, ones, ones, decay)[0], leaf, d)[0] for d in (lazy, plain)]
        assert torch.equal(*grads)
        lazy, plain = negated(6, width)
        w = torch.ones(width, device="cuda")
        for i in range(3):
            args, want = [torch.ones(6, width, device="cuda") for _ in range(3)], [torch.ones(6, width, device="cuda") for _ in range(3)]
            args[i], want[i] = lazy, plain
            assert all(torch.equal(a, b) for a, b in zip(ops.gated_residual_norm(*args, w, w, w), ops.gated_residual_norm(*want, w, w, w)))
