"""What is beyond the operators' limits raises ValueError like every call that cannot be right, and the entries of the library have the same
limits."""
import ctypes as C
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from rl4mm_amd import _lib, _policy_capi as capi, policy_ops as ops


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield lambda *shape, dtype=torch.float32, device="cuda", grad=False: torch.empty(*shape, dtype=dtype, device=device, requires_grad=grad)


def segment(fake, N, H, **kw):
    return ops.decay_attention(fake(2, N, H, 1), fake(2, N, H, 1), fake(2, N, H, 1), fake(H), **kw)


def step(fake, N, H, **kw):
    return ops.decay_attention_step(fake(N, H, 1), fake(N, H, 1), fake(N, H, 1), fake(H), fake(N, H, 1, 1), **kw)


@pytest.mark.parametrize("call", [segment, step])
@pytest.mark.parametrize("N, H", [(2**21 + 1, 2), (2**22 + 1, 1), (1, 2**16 + 1), (1000, 5000)], ids=str)
def test_units(fake, call, N, H):
    with pytest.raises(ValueError, match="environments of"):
        call(fake, N, H)


@pytest.mark.parametrize("call", [segment, step])
@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, math.inf, math.nan])
def test_scale(fake, call, scale):
    with pytest.raises(ValueError, match="32 bits"):
        call(fake, 2, 2, scale=scale)


@pytest.mark.parametrize("eps", [1e39, math.inf, 1e-39, -1.0])
def test_eps(fake, eps):
    with pytest.raises(ValueError, match="eps"):
        ops.gated_residual_norm(fake(2, 4), fake(2, 4), None, fake(4), fake(4), fake(4), eps)


def test_gradients(fake):
    with pytest.raises(ValueError, match="at most"):
        ops.clip_grad_norm([fake(1)] * (capi.MAX_TENSORS + 1), 1.0)


@pytest.mark.gpu
def test_sparse_gradients():
    """a CSR gradient has no strides to ask for: refused like any other layout"""
    for g in (torch.eye(3, device="cuda").to_sparse_csr(), torch.eye(3, device="cuda").to_sparse()):
        with pytest.raises(ValueError, match="strided"):
            ops.clip_grad_norm([torch.ones(3, device="cuda"), g], 1.0)


def test_the_entries_have_these_limits():
    lib = _lib.policy_binding()
    a = capi.Attention(heads=1, dk=1, dv=1, steps=1, envs=capi.MAX_UNITS, scale=1.0, log_decay=64)
    need = lib.fn["attention_workspace"]
    assert need(C.byref(a)) >= 0
    a.envs += 1
    assert need(C.byref(a)) == -1
    a.envs, a.heads = 1, capi.MAX_HEADS
    assert need(C.byref(a)) >= 0
    a.heads += 1
    assert need(C.byref(a)) == -1
    counts, dtypes = (C.c_int64 * (capi.MAX_TENSORS + 1))(), (C.c_int32 * (capi.MAX_TENSORS + 1))()
    assert lib.fn["clip_workspace"](counts, dtypes, capi.MAX_TENSORS) == 0 and lib.fn["clip_workspace"](counts, dtypes, capi.MAX_TENSORS + 1) == -1
