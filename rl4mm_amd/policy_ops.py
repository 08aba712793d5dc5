"""Operators for a policy that remembers order flow, as hand-written HIP kernels (include/lobpolicy.h): torch tensors in and out, launched
asynchronously on torch's current stream of the tensors' device, like the tensor path of rl4mm_amd/env.py they run next to.

  decay_attention_step   one observation of every environment: the state of each, [heads][dk][dv], is updated in place
  decay_attention        the same over recorded segments [T, N], differentiable
  gated_residual_norm    a block's end: norm, gate, residual scale, and the norm before the next block; differentiable
  clip_grad_norm         the global gradient norm, and clipping by it

float32 and bfloat16; states, norms and sums are float32 or wider, and a bfloat16 result is rounded once, as it is stored.  There is no CPU path: CPU tensors raise, as does a missing
library.  Every call can be captured into a graph (nothing waits for the device, nothing is allocated but results and workspaces, through
torch's allocator); a forward and a backward pass belong into the same capture, with no eager graph of the same leaves alive beside it, as torch
asks of every operation.  torch.compile runs them between its graphs; forward-mode differentiation, torch.jit.trace and make_fx, which cannot see a
launch, are refused.  A call that cannot be right raises ValueError or TypeError before anything is launched."""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from . import _policy_capi as capi

_DTYPES = {torch.float32: capi.F32, torch.bfloat16: capi.BF16}
_LARGEST = 2.0**128 - 2.0**104  # of the numbers of 32 bits


_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(index).cuda_stream without the object around it


_current_device = torch._C._cuda_getDevice


class _on:
    """The raw current stream of a device that is not the current one, with that device current inside the block."""

    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        torch.cuda.set_device(self.before)


def _call(device, name, *args):
    """An entry point of the library, on the current stream of `device`, which is made the current device for it."""
    lib = _lib._policy_binding or _lib.policy_binding()
    index = device.index
    if index == _current_device():
        code = lib.fn[name](*args, _raw_stream(index))
    else:
        with _on(index) as stream:
            code = lib.fn[name](*args, stream)
    if code < 0:
        lib.check(code, name)


_tracing, _modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
# the recorders that see operations before they are dispatched: the list itself, as looking it up takes longer than the rest of the check
_early_modes = next((v for k, v in vars(torch._ops.mode_stack_state_for_pre_dispatch()).items() if k.endswith("infra_modes")), [])
_NO_EARLY_MODES = [None] * len(_early_modes)


def _seen(*tensors):
    """Refuses what would pass the launches by without a word: tensors that carry a tangent, and recorders of torch's operations, whose record would lack them.
    (torch.compile runs the operators as they are, between its graphs.)"""
    if not _tracing() and not _modes() and _early_modes == _NO_EARLY_MODES and forward_ad._current_level < 0:
        return
    from torch._subclasses.fake_tensor import FakeTensor
    from torch.fx.experimental.proxy_tensor import get_proxy_mode

    _need(not _tracing(), "torch.jit.trace cannot record this operator: its launch would be missing from the trace")
    _need(get_proxy_mode() is None, "make_fx cannot record this operator: its launch would be missing from the graph")
    for t in tensors:
        if t is not None:
            _need(not isinstance(t, FakeTensor), "a fake tensor holds nothing to compute with", TypeError)
            _need(forward_ad._current_level < 0 or forward_ad.unpack_dual(t).tangent is None, "forward-mode differentiation is not there: a tangent would be lost")


def _new(t):
    """An empty tensor of t's shape and type, without gaps."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _need(ok, message, kind=ValueError):
    if not ok:
        raise kind(message)


def _tensor(t, name, dtypes, device=None, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is a torch tensor, got {type(t).__name__}")
    if not t.is_cuda or t.layout != torch.strided:
        raise ValueError(f"{name} is a strided tensor on the GPU (there is no CPU path): got {t.layout} on {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} is {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other operands on {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has the shape {tuple(shape)}, got {tuple(t.shape)}")


def _lined(t):
    """`t`, its last dimension contiguous, and its memory what it says (the imaginary part of a conjugate is negated on the way, unless it has been copied)."""
    return t.resolve_neg() if t.shape[-1] == 1 else t if t.stride(-1) == 1 else t.contiguous()


def _operand(t):  # [T, N, H, D] or [N, H, D]
    st = t.stride()
    return capi.Operand(t.data_ptr(), st[0], st[1], st[2]) if len(st) == 4 else capi.Operand(t.data_ptr(), 0, st[0], st[1])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _changed(tensors):
    """Tells autograd that these were written in place (tensors made in inference mode keep no count of it)."""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _flags(t, name, shape, device):
    if t is None or (type(t) is torch.Tensor and t.dtype is torch.bool and t.device == device and t.shape == shape and t.layout is torch.strided):
        return t
    _tensor(t, name, (torch.bool, torch.uint8), device, shape)
    return t


def _heads(q, k, v, log_decay, state, scale, dims):
    """Checks what the two forms have in common -> (log_decay, scale)."""
    try:  # one look at all of it; what is wrong is found out below
        device, shape = q.device, q.shape
        heads, dk, dv = shape[-2], shape[-1], v.shape[-1]
        fine = (
            q.is_cuda and q.dtype in _DTYPES and q.layout is torch.strided and len(shape) == len(dims) and heads >= 1 and 1 <= dk <= capi.MAX_HEAD and 1 <= dv <= capi.MAX_HEAD
            and k.dtype is q.dtype and k.device == device and k.shape == shape and k.layout is torch.strided
            and v.dtype is q.dtype and v.device == device and v.shape[:-1] == shape[:-1] and v.layout is torch.strided
            and log_decay.dtype is torch.float32 and log_decay.device == device and log_decay.shape == (heads,) and log_decay.is_contiguous() and not log_decay.requires_grad
            and (state is None or (state.dtype is torch.float32 and state.device == device and state.shape == (shape[-3], heads, dk, dv) and state.layout is torch.strided))
        )  # fmt: skip
    except (AttributeError, IndexError, TypeError):
        fine = False
    if not fine:
        _tensor(q, "q", _DTYPES)
        _need(q.dim() == len(dims), f"q is [{', '.join(dims)}], got {tuple(q.shape)}")
        _tensor(k, "k", (q.dtype,), q.device, q.shape)
        _tensor(v, "v", (q.dtype,), q.device)
        _need(v.shape[:-1] == q.shape[:-1], f"v is [{', '.join(dims[:-1])}, dv] beside q {tuple(q.shape)}, got {tuple(v.shape)}")
        shape, heads, dk, dv = q.shape, q.shape[-2], q.shape[-1], v.shape[-1]
        _need(heads >= 1 and 1 <= dk <= capi.MAX_HEAD and 1 <= dv <= capi.MAX_HEAD, f"{heads} heads of dk = {dk} and dv = {dv}: one head or more, dk and dv 1 to {capi.MAX_HEAD}")
        _tensor(log_decay, "log_decay", (torch.float32,), q.device, (heads,))
        _need(not log_decay.requires_grad, "log_decay takes no gradient: the decays are constants of the policy")
        if state is not None:
            _tensor(state, "the state", (torch.float32,), q.device, (q.shape[-3], heads, dk, dv))
        log_decay = log_decay.contiguous()
    _need(heads <= capi.MAX_HEADS and shape[-3] * heads <= capi.MAX_UNITS, f"{shape[-3]} environments of {heads} heads: heads to {capi.MAX_HEADS}, environments x heads to {capi.MAX_UNITS}")
    scale = dk**-0.5 if scale is None else float(scale)
    _need(abs(scale) <= _LARGEST, f"the scale {scale} is not finite in 32 bits")
    return log_decay, scale


def _describe(q, k, v, log_decay, reset, lengths, scale):
    a = capi.Attention()
    a.dtype, a.heads, a.dk, a.dv, a.envs, a.steps = _DTYPES[q.dtype], q.shape[-2], q.shape[-1], v.shape[-1], q.shape[-3], q.shape[0] if q.dim() == 4 else 1
    a.q, a.k, a.v = _operand(q), _operand(k), _operand(v)
    a.log_decay, a.scale = log_decay.data_ptr(), scale
    if reset is not None:
        a.reset = reset.data_ptr()
        a.reset_stride_t, a.reset_stride_n = reset.stride() if reset.dim() == 2 else (0, reset.stride(0))
    if lengths is not None:
        a.lengths = lengths.data_ptr()
    return a


def _workspace(a, lib, device):
    """The description's workspace -> the tensor that holds it (to be kept until the launch is made), or None."""
    need = lib.check(lib.fn["attention_workspace"](C.byref(a)), "attention_workspace")
    held = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    a.workspace, a.workspace_bytes = _ptr(held), need
    return held


def _attention_forward(q, k, v, log_decay, state, reset, lengths, scale):
    out = _new(v)
    last = torch.empty((q.shape[1], q.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32, device=q.device)
    lib = _lib.policy_binding()
    a = _describe(q, k, v, log_decay, reset, lengths, scale)
    a.out, a.state_in, a.state_out = _operand(out), _ptr(state), last.data_ptr()
    held = _workspace(a, lib, q.device)
    _call(q.device, "attention_forward", C.byref(a))
    return out, last, held


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, reset, lengths, scale):
        ctx.set_materialize_grads(False)
        out, last, held = _attention_forward(q, k, v, log_decay, state, reset, lengths, scale)
        ctx.save_for_backward(q, k, v, log_decay, state, reset, lengths, held)
        ctx.scale = scale
        return out, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlast):
        q, k, v, log_decay, state, reset, lengths, forward = ctx.saved_tensors
        if dout is None and dlast is None:
            return (None,) * 8
        dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if dout is None else _lined(dout)
        dlast = None if dlast is None else dlast.contiguous()
        dq, dk, dv = _new(q), _new(k), _new(v)
        dstate = _new(state) if ctx.needs_input_grad[4] else None
        lib = _lib.policy_binding()
        a = _describe(q, k, v, log_decay, reset, lengths, ctx.scale)
        a.out, a.state_in, a.grad_state_out = _operand(dout), _ptr(state), _ptr(dlast)
        a.grad_q, a.grad_k, a.grad_v, a.grad_state_in = _operand(dq), _operand(dk), _operand(dv), _ptr(dstate)
        held = _workspace(a, lib, q.device)  # noqa: F841
        a.forward_workspace = _ptr(forward)
        _call(q.device, "attention_backward", C.byref(a))
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, dstate, None, None, None


def decay_attention(q, k, v, log_decay, *, initial_state=None, reset=None, lengths=None, scale=None):
    """Linear attention with a decay for each head over recorded segments -> (out [T, N, H, dv], state [N, H, dk, dv] after the last token).

    Of every environment n and head h, with a state S [dk, dv] that begins as ``initial_state`` (zeros without one):

        S = 0 where reset[t, n];   S = exp(log_decay[h]) S + k_t v_t^T;   out_t = scale q_t^T S

    q, k [T, N, H, dk], v [T, N, H, dv], float32 or bfloat16, time-major like the framework's traces; any strides, so they may be views of one
    projection's output.  log_decay [H] float32, a constant (no gradient).  reset [T, N] bool or uint8: token t is the first of a new episode, and
    nothing before it reaches it - not even a value that is not a number.  lengths [N] int32: environment n has that many tokens (clamped to 0 .. T);
    what lies behind them is not used, its rows of ``out`` and of the gradients are 0, and the state is the one after its last token.  scale: dk ** -0.5
    by default.  Gradients reach q, k, v and initial_state.  bfloat16: what lies between the operands and a result is held in 32 bits, or in two
    bfloat16 that are off by 2^-16 of a term; decays are float32 exponentials, off by 2^-24 of them and of their exponent."""
    log_decay, scale = _heads(q, k, v, log_decay, initial_state, scale, ("T", "N", "H", "dk"))
    reset = _flags(reset, "reset", q.shape[:2], q.device)
    if lengths is not None:
        _tensor(lengths, "lengths", (torch.int32,), q.device, (q.shape[1],))
        lengths = lengths.contiguous()
    _seen(q, k, v, log_decay, initial_state)
    if q.shape[0] == 0 or q.shape[1] == 0:  # (nothing to compute, and the gradients of what is empty are zeros: torch's own operations say so)
        state = torch.zeros((*q.shape[1:], v.shape[3]), dtype=torch.float32, device=q.device) if initial_state is None else initial_state
        nothing = 0.0 * (q.sum() + k.sum() + v.sum())
        return v + nothing + 0.0 * state.sum().to(v.dtype), state + nothing.float()
    state = None if initial_state is None else initial_state.contiguous()
    args = (_lined(q), _lined(k), _lined(v), log_decay, state, reset, lengths, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        return _DecayAttention.apply(*args)
    return _attention_forward(*args)[:2]


def decay_attention_step(q, k, v, log_decay, state, *, reset=None, skip=None, scale=None):
    """One token of every environment -> out [N, H, dv]; ``state`` [N, H, dk, dv] float32, contiguous, is updated IN PLACE.

    The step of ``decay_attention`` (q, k [N, H, dk], v [N, H, dv]): reset [N] - this observation begins an episode; skip [N] - the environment is
    done and sits out (the ``done`` flags of ``vector_step_tensors``): its state stays as it is, its row of out is 0.  No gradient: raises when one
    is asked for."""
    log_decay, scale = _heads(q, k, v, log_decay, state, scale, ("N", "H", "dk"))
    _need(state is not None, "state is the [N, H, dk, dv] tensor that the step updates", TypeError)
    _need(state.is_contiguous(), "the state is updated in place: it has to be contiguous")
    _need(not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad)),
          "decay_attention_step has no gradient: call it under torch.no_grad(), or decay_attention for the gradients")  # fmt: skip
    reset, skip = _flags(reset, "reset", q.shape[:1], q.device), _flags(skip, "skip", q.shape[:1], q.device)
    _seen(q, k, v, log_decay, state)
    out = _new(v)
    if q.shape[0] == 0:
        return out
    q, k, v = _lined(q), _lined(k), _lined(v)
    skip = None if skip is None else skip.contiguous()
    a = _describe(q, k, v, log_decay, reset, None, scale)
    a.out, a.state_out, a.skip = _operand(out), state.data_ptr(), _ptr(skip)
    _call(q.device, "attention_step", C.byref(a))
    _changed([state])
    return out


# ---- the block's end ----------------------------------------------------------------------------------------------------------


def _rows(t, width):
    """[..., width] -> [rows, width] with contiguous rows; a copy only where the strides leave no other way."""
    t = _lined(t)
    return t if t.dim() == 2 else t.reshape(-1, width)


def _describe_block(x, block, gate, post, res, pre, eps):
    b = capi.Block()
    b.stream_dtype, b.dtype, b.rows, b.width = _DTYPES[x.dtype], _DTYPES[block.dtype], *x.shape
    b.x, b.block, b.gate, b.x_stride, b.block_stride = x.data_ptr(), block.data_ptr(), _ptr(gate), x.stride(0), block.stride(0)
    b.gate_stride = 0 if gate is None else gate.stride(0)
    b.post, b.res, b.pre, b.eps = post.data_ptr(), res.data_ptr(), pre.data_ptr(), eps
    return b


def _block_forward(x, block, gate, post, res, pre, eps):
    y, z = _new(x), _new(block)
    b = _describe_block(x, block, gate, post, res, pre, eps)
    b.y, b.z = y.data_ptr(), z.data_ptr()
    _call(x.device, "block_forward", C.byref(b))
    return y, z


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, gate, post, res, pre, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, block, gate, post, res, pre)
        ctx.eps = eps
        return _block_forward(x, block, gate, post, res, pre, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz):
        x, block, gate, post, res, pre = ctx.saved_tensors
        if dy is None and dz is None:
            return (None,) * 7
        dy, dz = (None if d is None else _lined(d) for d in (dy, dz))
        dx, dblock = _new(x), _new(block)
        dgate = None if gate is None else _new(block)
        dpost, dres, dpre = _new(post), _new(res), _new(pre)
        lib = _lib.policy_binding()
        b = _describe_block(x, block, gate, post, res, pre, ctx.eps)
        b.grad_y, b.grad_z = _ptr(dy), _ptr(dz)
        b.grad_y_stride, b.grad_z_stride = 0 if dy is None else dy.stride(0), 0 if dz is None else dz.stride(0)
        b.grad_x, b.grad_block, b.grad_gate = dx.data_ptr(), dblock.data_ptr(), _ptr(dgate)
        b.grad_post, b.grad_res, b.grad_pre = dpost.data_ptr(), dres.data_ptr(), dpre.data_ptr()
        need = lib.check(lib.fn["block_workspace"](C.byref(b)), "block_workspace")
        held = torch.empty(need, dtype=torch.uint8, device=x.device)
        b.workspace, b.workspace_bytes = held.data_ptr(), need
        _call(x.device, "block_backward", C.byref(b))
        return tuple(g if wanted else None for g, wanted in zip((dx, dblock, dgate, dpost, dres, dpre), ctx.needs_input_grad)) + (None,)


def gated_residual_norm(x, block, gate, post_weight, residual_scale, pre_weight, eps=1e-6):
    """A block's end and the next one's beginning -> (y, z), both shaped like x [..., width]:

        y = x + residual_scale * sigmoid(gate) * post_weight * block / rms(block);   z = pre_weight * y / rms(y);   rms(a) = sqrt(mean(a ** 2) + eps)

    x: the residual stream, float32 or bfloat16, y its type.  block: what the block put out; gate: its gate's logits (None: no gate); z has their type,
    float32 or bfloat16, and is taken from y before that is rounded.  The three weights: float32 [width].  width: 1 to 8192; rows of any stride.
    Differentiable in all six; the weights' gradients are summed in a fixed order.  The gate's exponential and reciprocal are the hardware's: off by about
    (1 + abs(gate)) 2^-23 of sigmoid(gate) and of its slope, however far open or shut the gate is."""
    weights = (post_weight, residual_scale, pre_weight)
    try:  # one look at all of it; what is wrong is found out below
        device, shape = x.device, x.shape
        width = shape[-1]
        fine = (
            x.is_cuda and x.dtype in _DTYPES and x.layout is torch.strided and 1 <= width <= capi.MAX_WIDTH
            and block.dtype in _DTYPES and block.device == device and block.shape == shape and block.layout is torch.strided
            and (gate is None or (gate.dtype is block.dtype and gate.device == device and gate.shape == shape and gate.layout is torch.strided))
            and all(w.dtype is torch.float32 and w.device == device and w.shape == (width,) for w in weights)
        )  # fmt: skip
    except (AttributeError, IndexError, TypeError):
        fine = False
    if not fine:
        _tensor(x, "x", _DTYPES)
        _need(x.dim() >= 1, "x is [..., width], got a single number")
        width = x.shape[-1]
        _need(1 <= width <= capi.MAX_WIDTH, f"width = {width}: 1 to {capi.MAX_WIDTH}")
        _tensor(block, "block", _DTYPES, x.device, x.shape)
        if gate is not None:
            _tensor(gate, "gate", (block.dtype,), x.device, x.shape)
        for t, name in zip(weights, ("post_weight", "residual_scale", "pre_weight")):
            _tensor(t, name, (torch.float32,), x.device, (width,))
    eps = float(eps)
    _need(2.0**-126 <= eps <= _LARGEST, "eps is a positive number that 32 bits hold")
    _seen(x, block, gate, *weights)
    shape, wanted = x.shape, torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, block, gate, *weights))
    rows = [_rows(t, width) if t is not None else None for t in (x, block, gate)]
    if x.numel() == 0:  # (nothing to compute, and the gradients are zeros: torch's own operations say so)
        nothing = 0.0 * sum(t.sum().float() for t in (*rows, *weights) if t is not None)
        return tuple((t + nothing).to(t.dtype).reshape(shape) for t in rows[:2])
    args = (*rows, *(t.contiguous() for t in weights), eps)
    y, z = _GatedResidualNorm.apply(*args) if wanted else _block_forward(*args)
    return (y, z) if len(shape) == 2 else (y.view(shape), z.view(shape))


# ---- the global gradient norm -------------------------------------------------------------------------------------------------


def _dense(t):
    """Whether t's elements fill its span of memory once each, in whatever order."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def clip_grad_norm(grads, max_norm, norm_type=2.0):
    """Scales ``grads`` IN PLACE by min(1, max_norm / (norm + 1e-6)) -> norm, one float32 on their device (nothing waits for it).

    grads: a tensor, or an iterable of tensors (None among them is passed over: a parameter without a gradient); float32 and bfloat16, mixed as you like, on
    one GPU, each dense in some order of its dimensions, no two of them overlapping.  norm_type 2.0: the root of the sum of all squares, summed in 64 bits
    in a fixed order; float("inf"): the largest magnitude.  A gradient that is not a number makes the norm one, and with it every gradient; an infinite
    norm makes the finite ones 0 (and with an infinite max_norm all of them not numbers, as the quotient is none).  No gradients: the norm is a CPU zero, as there is no device to put it on."""
    grads = [grads] if isinstance(grads, torch.Tensor) else [g for g in grads if g is not None]
    max_norm, norm_type = float(max_norm), float(norm_type)
    _need(max_norm >= 0.0, f"max_norm = {max_norm}: 0 or more")
    _need(norm_type in (2.0, math.inf), f"norm_type = {norm_type}: 2 or inf")
    if not grads:
        return torch.zeros(())
    _need(len(grads) <= capi.MAX_TENSORS, f"{len(grads)} gradients: {capi.MAX_TENSORS} at most")
    device, spans = getattr(grads[0], "device", None), []
    for i, g in enumerate(grads):
        if not (type(g) is torch.Tensor and g.dtype in _DTYPES and g.device == device and g.is_cuda and not g.requires_grad and g.layout is torch.strided and g.is_contiguous()):
            _tensor(g, f"gradient {i}", _DTYPES, device)
            _need(not g.requires_grad, f"gradient {i} requires a gradient itself: it is scaled outside autograd (detach it)")
            _need(_dense(g), f"gradient {i} is not dense in memory (shape {tuple(g.shape)}, strides {g.stride()}): it could not be scaled in place")
        count = g.numel()
        if count:
            spans.append((g.data_ptr(), count * g.itemsize, i))
    spans.sort()
    end, last = 0, -1
    for p, size, i in spans:
        if p < end:
            raise ValueError(f"gradients {min(i, last)} and {max(i, last)} share memory: each element is counted and scaled once")
        end, last = p + size, i
    _seen(*grads)
    n = len(grads)
    tensors = (C.c_void_p * n)(*[g.data_ptr() for g in grads])
    counts, dtypes = (C.c_int64 * n)(*[g.numel() for g in grads]), (C.c_int32 * n)(*[_DTYPES[g.dtype] for g in grads])
    lib = _lib.policy_binding()
    need = lib.check(lib.fn["clip_workspace"](counts, dtypes, n), "clip_workspace")
    norm, held = torch.empty((), dtype=torch.float32, device=device), torch.empty(max(need, 8), dtype=torch.uint8, device=device)
    _call(device, "clip", tensors, counts, dtypes, n, 2 if norm_type == 2.0 else 0, max_norm, norm.data_ptr(), held.data_ptr(), need)
    _changed(grads)
    return norm
