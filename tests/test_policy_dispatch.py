"""Which agents summary.generate_trajectories runs as a sequence policy."""
import types

import numpy as np
import pytest

from rl4mm_amd import summary
from rl4mm_amd.agents import FixedActionAgent, Teradactyl


class Venv:
    num_envs, episode_length, step_size = 2, 4.0, 1.0
    sim = types.SimpleNamespace(action_dim=4)

    def vector_reset(self):
        pass


class Remembers(FixedActionAgent):
    """a rule-based agent with attributes of its own"""

    memory = None

    def act(self, *a):
        raise AssertionError

    def remember(self):
        return self.memory


class Policy:
    def memory(self, envs):
        return []

    def act(self, observations, memory, reset=None, skip=None):
        return None


class Other:
    memory = act = 3


@pytest.mark.parametrize("agent, as_policy", [(Policy(), True), (Remembers(np.ones(4)), False), (type("Both", (Policy, FixedActionAgent), {})(np.ones(4)), False), (Other(), False), (object(), False)],
                         ids=["a policy", "rule-based, remembers", "rule-based, both methods", "attributes", "neither"])  # fmt: skip
def test_which(monkeypatch, agent, as_policy):
    class Policies(Exception):
        pass

    class Rules(Exception):
        pass

    def raises(kind):
        def f(*a):
            raise kind

        return f

    monkeypatch.setattr(summary, "_policy_trajectories", raises(Policies))
    if isinstance(agent, (FixedActionAgent, Teradactyl)):
        monkeypatch.setattr(summary, "policy_of", raises(Rules))
    with pytest.raises(Policies if as_policy else Rules if isinstance(agent, FixedActionAgent) else TypeError):
        summary.generate_trajectories(agent, Venv())
