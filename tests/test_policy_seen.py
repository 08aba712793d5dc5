"""Forward-mode differentiation and recorders of torch's operations cannot see the operators' launches: each entry refuses them rather than let a tangent, or
itself, get lost.  Without a GPU: the checks of devices and the launches are stubbed out."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from rl4mm_amd import policy_ops as ops


pytestmark = pytest.mark.filterwarnings("ignore")  # (the tracers' own)


@pytest.fixture
def calls(monkeypatch):
    """entry -> (function of one operand, that operand); the launches are recorded, not made"""
    launched = []
    monkeypatch.setattr(ops, "_tensor", lambda *a, **k: None)
    monkeypatch.setattr(ops, "_call", lambda device, name, *args: launched.append(name))

    class Library:
        fn = {name: (lambda *a: 64) for name in ("attention_workspace", "block_workspace", "clip_workspace")}

        def check(self, code, what):
            return code

    monkeypatch.setattr(ops._lib, "policy_binding", Library)
    q, v, g, state, w = torch.ones(4, 3, 2, 8), torch.ones(4, 3, 2, 8), torch.zeros(2), torch.zeros(3, 2, 8, 8), torch.ones(8)
    return launched, {
        "segment": (lambda t: ops.decay_attention(t, q, v, g)[0], q),
        "segment's state": (lambda t: ops.decay_attention(q, q, v, g, initial_state=t)[1], state),
        "step": (lambda t: ops.decay_attention_step(t, q[0], v[0], g, state), q[0]),
        "step's state": (lambda t: ops.decay_attention_step(q[0], q[0], v[0], g, t), state),
        "block": (lambda t: ops.gated_residual_norm(t, v, None, w, w, w)[0], v),
        "block's weight": (lambda t: ops.gated_residual_norm(v, v, None, w, w, t)[1], w),
        "clip": (lambda t: ops.clip_grad_norm([t], 1.0), w.clone()),
    }


ENTRIES = ["segment", "segment's state", "step", "step's state", "block", "block's weight", "clip"]


@pytest.mark.parametrize("entry", ENTRIES)
def test_tangents(calls, entry):
    launched, (f, x) = calls[0], calls[1][entry]
    with fw.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            f(fw.make_dual(x, torch.ones_like(x)))
        assert not launched
        f(x)  # (no tangent: a call like any other)
    assert launched


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("record", [lambda f, x: torch.jit.trace(f, (x,), check_trace=False), lambda f, x: make_fx(f)(x), lambda f, x: make_fx(f, pre_dispatch=True)(x)], ids=["jit", "fx", "fx before dispatch"])
def test_recorders(calls, entry, record):
    launched, (f, x) = calls[0], calls[1][entry]
    with pytest.raises(ValueError, match="cannot record"):
        record(f, x)
    assert not launched


@pytest.mark.parametrize("entry", ENTRIES)
def test_fake_tensors(calls, entry):
    launched, (f, x) = calls[0], calls[1][entry]
    mode = FakeTensorMode(allow_non_fake_inputs=True)
    with mode, pytest.raises(TypeError, match="fake"):
        f(mode.from_tensor(x))
    assert not launched


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("around", [contextlib.nullcontext, torch.no_grad, torch.inference_mode, lambda: FlopCounterMode(display=False), lambda: torch.autocast("cpu", torch.bfloat16)],
                         ids=["nothing", "no_grad", "inference", "a counter", "autocast"])  # fmt: skip
def test_other_surroundings(calls, entry, around):
    launched, (f, x) = calls[0], calls[1][entry]
    with around():
        f(x)
    assert launched


@pytest.mark.gpu
def test_between_compiled_graphs():
    """torch.compile runs the operators as they are: the results and gradients of the plain calls."""
    from test_gpu_policy_ops import F32, block_problem, problem

    p, dout, dlast = problem(1, 50, 3, 2, 64, 64, F32, 0.05, True)
    args, dy, dz = block_problem(3, 24, 64, F32, F32)

    def segment(q, k, v, s):
        out, last = ops.decay_attention(q * 2, k, v, p["log_decay"], initial_state=s, reset=p["reset"], lengths=p["lengths"])
        return out + 1, last * 3

    def block(*a):
        y, z = ops.gated_residual_norm(*a)
        return y + 1, z * 2

    def trained(f, operands, grads):
        leaves = [t.detach().clone().requires_grad_(True) for t in operands]
        results = f(*leaves)
        return [*(r.detach() for r in results), *torch.autograd.grad(results, leaves, grads)]

    def step(q, k, v, s):
        return ops.decay_attention_step(q * 2, k, v, p["log_decay"], s) + 1, s * 1

    def clip(a, b):
        return ops.clip_grad_norm([a, b], 0.5) + 1, a * 1, b * 1

    qkvs = [p[key] for key in ("q", "k", "v", "state")]
    for run in (lambda f: trained(f(segment), qkvs, [dout, dlast]), lambda f: f(segment)(*qkvs), lambda f: trained(f(block), args, [dy, dz]),
                lambda f: f(step)(*(t[0] for t in qkvs[:3]), qkvs[3].clone()), lambda f: f(clip)(args[0].clone(), args[1].clone())):  # fmt: skip
        torch._dynamo.reset()
        for want, got in zip(run(lambda f: f), run(lambda f: torch.compile(f, backend="eager"))):
            assert torch.equal(want, got)
