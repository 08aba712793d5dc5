"""Recorded segments padded with anything: what lies behind an environment's last step reaches no gradient of a SequencePolicy.  On the CPU with plain
stand-ins for the two operators, on the GPU with the operators."""
import math

import numpy as np
import pytest
import torch

from rl4mm_amd import policy as P
import policy_reference as ref

T, N, D = 40, 5, 6
LENGTHS = [40, 17, 0, 39, 1]


def make(device):
    torch.manual_seed(3)
    return P.SequencePolicy(np.full(D, -2.0), np.full(D, 3.0), np.full(4, 10.0), width=96, blocks=2, heads=3, head_dim=32).to(device)


def attention(q, k, v, log_decay, *, initial_state=None, reset=None, lengths=None, scale=None):
    """plain torch, differentiable: the matrix of weights of each environment"""
    gap = torch.arange(q.shape[0])[:, None] - torch.arange(q.shape[0])[None]
    there = torch.arange(q.shape[0])[:, None] < lengths[None]
    q, k, v = (torch.where(there[..., None, None], t, torch.zeros(())).permute(1, 2, 0, 3) for t in (q, k, v))
    weight = torch.where(gap >= 0, torch.exp(log_decay[:, None, None] * gap.clamp(min=0)), torch.zeros(()))
    out = ((q @ k.transpose(-1, -2) * weight) @ v * q.shape[-1] ** -0.5).permute(2, 0, 1, 3)
    return torch.where(there[..., None, None], out, torch.zeros(())), None


def block(x, b, gate, post, res, pre, eps):
    rms = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)  # noqa: E731
    y = x + res * torch.sigmoid(gate) * post * rms(b)
    return y, pre * rms(y)


def gradients(policy, observations, lengths):
    actions, values, _ = policy(observations, lengths=lengths)
    assert torch.isfinite(actions).all() and torch.isfinite(values).all()
    there = torch.arange(T, device=lengths.device)[:, None] < lengths
    loss = (actions[there].square().sum() + (values[there] - 1.0).square().sum()) / there.sum()
    return [loss.detach(), actions[there].detach()] + list(torch.autograd.grad(loss, list(policy.parameters())))


def compare(policy, junk, dtype, device):
    gen = torch.Generator().manual_seed(1)
    clean = torch.randn(T, N, D, generator=gen, dtype=dtype)
    lengths = torch.tensor(LENGTHS, dtype=torch.int32)
    dirty = torch.where((torch.arange(T)[:, None] >= lengths)[..., None], torch.full((), junk, dtype=dtype), clean)
    want, got = (gradients(policy, o.to(device), lengths.to(device)) for o in (clean, dirty))
    for w, g in zip(want, got):
        assert torch.isfinite(g).all() and torch.equal(w, g)  # (a gradient of 0 times any finite number adds 0)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf, 1e38, -1e30])
def test_padding_with_stand_ins(monkeypatch, junk, dtype):
    monkeypatch.setattr(P.ops, "decay_attention", attention)
    monkeypatch.setattr(P.ops, "gated_residual_norm", block)
    compare(make("cpu"), junk, dtype, "cpu")


def test_stand_in_is_the_operator():
    gen = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(9, 3, 2, 4, generator=gen, dtype=torch.float64) for _ in range(3))
    g, lengths = torch.tensor([-0.3, -0.01]), torch.tensor([9, 4, 0])
    assert torch.allclose(attention(q, k, v, g.double(), lengths=lengths)[0], ref.attention(q, k, v, g, lengths=lengths, scale=0.5)["out"], rtol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf, 1e38, -1e30])
def test_padding(junk, dtype):
    compare(make("cuda"), junk, dtype, "cuda")


@pytest.mark.gpu
def test_an_update_on_padded_segments():
    """and the update that follows leaves every parameter a number"""
    policy = make("cuda")
    observations = torch.randn(T, N, D, generator=torch.Generator().manual_seed(4), dtype=torch.float64).cuda()
    lengths = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda")
    there = torch.arange(T, device="cuda")[:, None] < lengths
    observations[~there] = math.nan
    _, values, _ = policy(observations, lengths=lengths)
    norm = P.update(policy, torch.optim.SGD(policy.parameters(), lr=0.1), values[there].square().sum())
    assert torch.isfinite(norm) and all(torch.isfinite(p).all() for p in policy.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("lengths, error", [(torch.zeros(N + 1, dtype=torch.int32), ValueError), (torch.zeros(N, dtype=torch.int32), ValueError), (torch.zeros(N), TypeError), ([1] * N, TypeError)],
                         ids=["too many", "on the host", "type", "a list"])  # fmt: skip
def test_lengths_that_are_none(lengths, error):
    """refused by the operator, as without padding"""
    policy = make("cuda")
    if isinstance(lengths, torch.Tensor) and not (error is ValueError and len(lengths) == N):
        lengths = lengths.cuda()
    with pytest.raises(error):
        policy(torch.randn(T, N, D, device="cuda"), lengths=lengths)
