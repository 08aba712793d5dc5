"""A policy that remembers order flow: what an environment's observations so far mean for its next action, in a state per environment.

The reference's learner is an RLlib PPO whose policy sees one observation at a time (rl4mm/helpers/main_helper.py:253-300); what a quote should be
depends on what the book did before.  ``SequencePolicy`` keeps that in the states of decay attention (rl4mm_amd/policy_ops.py), in two forms that are
the same function:

  act       one step of every environment of a batch, on the tensors of ``HistoricalOrderbookVectorEnv.vector_step_tensors``: the memory is updated in
            place, forgotten where an episode begins, left alone where an environment is done
  forward   recorded segments [T, N] at once, differentiable: what an update trains on

Parameters and memories are float32; under ``torch.autocast("cuda", torch.bfloat16)`` the projections, and with them the operators, work in bfloat16.

``update`` takes a step of any torch optimizer with the gradients clipped by their global norm, and
``summary.generate_trajectories`` / ``get_episode_summary_dict`` evaluate the policy like the rule-based agents."""
from __future__ import annotations

import torch

from . import policy_ops as ops


class _Block(torch.nn.Module):
    def __init__(self, width, heads, head_dim):
        super().__init__()
        self.mix = torch.nn.Linear(width, 3 * heads * head_dim + width)  # queries, keys, values, and the gate of what comes out
        self.out = torch.nn.Linear(heads * head_dim, width)
        self.post = torch.nn.Parameter(torch.ones(width))
        self.scale = torch.nn.Parameter(torch.full((width,), 0.5))
        self.pre = torch.nn.Parameter(torch.ones(width))  # of the norm in front of the next block (or the heads)


class SequencePolicy(torch.nn.Module):
    """observation_low, observation_high: the bounds of the observation space (observations are scaled by them); action_high: the upper bound of each
    action, whose lower bound is 0 (the Beta parameters of a side's quotes, rl4mm/gym/HistoricalOrderbookEnvironment.py:85-94).  The memories' time scales
    are constants: ``shortest`` steps for the first head, twice as long from head to head."""

    def __init__(self, observation_low, observation_high, action_high, width=256, blocks=2, heads=4, head_dim=64, shortest=16.0, eps=1e-6):
        super().__init__()
        low, high = torch.as_tensor(observation_low, dtype=torch.float64), torch.as_tensor(observation_high, dtype=torch.float64)
        self.register_buffer("low", low.float())
        self.register_buffer("span", (high - low).clamp(min=1e-6).float())
        self.register_buffer("action_high", torch.as_tensor(action_high, dtype=torch.float64))
        if not shortest > 1.0:
            raise ValueError(f"shortest = {shortest}: the shortest memory lasts more than one step")
        self.register_buffer("log_decay", torch.log1p(-1.0 / (shortest * torch.exp2(torch.arange(heads, dtype=torch.float64)))).float())
        self.width, self.heads, self.head_dim, self.eps = width, heads, head_dim, eps
        self.embed = torch.nn.Linear(len(low), width)
        self.first = torch.nn.Parameter(torch.ones(width))
        self.blocks = torch.nn.ModuleList(_Block(width, heads, head_dim) for _ in range(blocks))
        self.action = torch.nn.Linear(width, len(self.action_high))
        self.value = torch.nn.Linear(width, 1)

    @classmethod
    def for_env(cls, venv, **kw):
        """The policy of a ``HistoricalOrderbookVectorEnv``'s spaces, on its device."""
        return cls(venv.observation_space.low, venv.observation_space.high, venv.action_space.high, **kw).to(torch.device("cuda", venv.sim.cfg.device_id))

    def memory(self, envs):
        """The empty memory of ``envs`` environments: a state per block."""
        return [torch.zeros(envs, self.heads, self.head_dim, self.head_dim, dtype=torch.float32, device=self.log_decay.device) for _ in self.blocks]

    def _walk(self, observations, attend, behind=None):
        scaled = (observations.float() - self.low) / self.span
        if behind is not None:  # (times a gradient of 0, what is not finite or overflows on its way would be a gradient that is no number)
            scaled = torch.where(behind[..., None], scaled.nan_to_num(0.0, 0.0, 0.0).clamp(-(2.0**16), 2.0**16), scaled)
        x = self.embed(scaled)
        z = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps) * self.first
        for i, block in enumerate(self.blocks):
            inner = self.heads * self.head_dim
            q, k, v, gate = block.mix(z).split([inner, inner, inner, self.width], dim=-1)
            q, k, v = (t.unflatten(-1, (self.heads, self.head_dim)) for t in (q, k, v))
            x, z = ops.gated_residual_norm(x, block.out(attend(i, q, k, v).flatten(-2)), gate, block.post, block.scale, block.pre, self.eps)
        return torch.sigmoid(self.action(z)).double() * self.action_high, self.value(z).squeeze(-1)

    @torch.no_grad()
    def act(self, observations, memory, reset=None, skip=None):
        """observations [N, D] -> actions float64 [N, A] in (0, action_high), as ``vector_step_tensors`` takes them.  ``memory`` (of ``memory(N)``) is updated
        in place; reset [N]: the observation begins an episode; skip [N] (the ``done`` flags): the environment sits out, its memory stays."""
        return self._walk(observations, lambda i, q, k, v: ops.decay_attention_step(q, k, v, self.log_decay, memory[i], reset=reset, skip=skip))[0]

    def forward(self, observations, memory=None, reset=None, lengths=None):
        """observations [T, N, D] -> (actions float64 [T, N, A], values [T, N], the memory after the last step): differentiable.  reset [T, N]: where
        episodes begin; lengths [N] int32: how many steps of each environment there are; memory: what came before (empty without one).  Behind an
        environment's last step the observations may hold anything; the actions and values there are finite and mean nothing: leave them out of the loss."""
        after = []
        behind = None
        if isinstance(lengths, torch.Tensor) and lengths.device == observations.device and lengths.shape == observations.shape[1:2]:  # (others the operator refuses)
            behind = torch.arange(observations.shape[0], device=observations.device)[:, None] >= lengths

        def attend(i, q, k, v):
            out, state = ops.decay_attention(q, k, v, self.log_decay, initial_state=None if memory is None else memory[i], reset=reset, lengths=lengths)
            after.append(state)
            return out

        actions, values = self._walk(observations, attend, behind)
        return actions, values, after


def update(policy, optimizer, loss, max_norm=0.5):
    """One step of ``optimizer`` down ``loss``'s gradient, clipped to the global norm ``max_norm`` -> the norm before clipping (on the device, unwaited for)."""
    optimizer.zero_grad(set_to_none=True)
    loss.backward()
    norm = ops.clip_grad_norm([p.grad for p in policy.parameters()], max_norm)
    optimizer.step()
    return norm
