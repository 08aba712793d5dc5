"""CPU-only: the policy operators' library builds for gfx950, exports what include/lobpolicy.h declares, and refuses what cannot be right before
anything is launched; the plain references' gradients are those of differences."""
import ctypes as C
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import policy_reference as ref
from rl4mm_amd import _capi, _lib, _policy_capi as capi, policy_ops as ops

ROOT = Path(__file__).resolve().parent.parent


def test_header_binding_and_library_agree():
    text = (ROOT / "include" / "lobpolicy.h").read_text()
    declared = set(re.findall(r"\b(lobpolicy_[a-z_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert declared == {"lobpolicy_" + n for n in capi.PROTOTYPES}
    assert set(_lib.policy_binding().fn) == set(capi.PROTOTYPES)


def test_struct_layouts(tmp_path):
    """The header's structs as the C compiler lays them out against the ctypes mirror."""
    lines = []
    for cname, cls in (("lobpolicy_operand", capi.Operand), ("lobpolicy_attention", capi.Attention), ("lobpolicy_block", capi.Block)):
        lines.append(f'_Static_assert(sizeof({cname}) == {C.sizeof(cls)}, "{cname}");')
        lines += [f'_Static_assert(offsetof({cname}, {f}) == {getattr(cls, f).offset}, "{cname}.{f}");' for f, _ in cls._fields_]
    lines.append(f'_Static_assert(LOBPOLICY_ABI_VERSION == {capi.ABI_VERSION} && LOBPOLICY_MAX_HEAD == {capi.MAX_HEAD} && LOBPOLICY_MAX_WIDTH == {capi.MAX_WIDTH}, "constants");')
    src = tmp_path / "sizes.c"
    src.write_text('#include <stddef.h>\n#include "lobpolicy.h"\n' + "\n".join(lines) + "\nint main(void) { return 0; }\n")
    subprocess.check_call(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(ROOT / "include"), "-c", str(src), "-o", str(tmp_path / "sizes.o")])


# ---- refusals at the C entries: a description that cannot be right returns before any launch ------------------------------------


def attention(**kw):
    a = capi.Attention()
    a.heads, a.dk, a.dv, a.steps, a.envs, a.scale = 2, 16, 16, 4, 3, 1.0
    a.log_decay = 64
    for key, value in kw.items():
        setattr(a, key, value)
    return a


@pytest.mark.parametrize("wrong", [dict(dtype=7), dict(dtype=-1), dict(heads=0), dict(heads=1 << 17), dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=129), dict(steps=0), dict(steps=1 << 31),
                                   dict(envs=0), dict(envs=1 << 30), dict(log_decay=None), {}])  # fmt: skip
def test_attention_entries_refuse(wrong):
    lib = _lib.policy_binding()
    a = attention(**wrong)
    for name in ("attention_forward", "attention_backward", "attention_step"):
        assert lib.fn[name](C.byref(a), None) == -1 and lib.fn["last_error"]()  # ({}: no operands)
    if wrong:
        assert lib.fn["attention_workspace"](C.byref(a)) == -1
    assert lib.fn["attention_forward"](None, None) == -1 and lib.fn["attention_workspace"](None) == -1
    with pytest.raises(_capi.LobsimError, match="attention_forward"):
        lib.check(lib.fn["attention_forward"](None, None), "attention_forward")


@pytest.mark.parametrize("wrong", [dict(dtype=3), dict(stream_dtype=2), dict(rows=0), dict(rows=1 << 41), dict(width=0), dict(width=8193), dict(x=None), dict(pre=None), {}])
def test_block_entries_refuse(wrong):
    lib = _lib.policy_binding()
    b = capi.Block()
    b.rows, b.width, b.eps = 4, 16, 1e-6
    b.x = b.block = b.post = b.res = b.pre = 64
    for key, value in wrong.items():
        setattr(b, key, value)
    for name in ("block_forward", "block_backward"):
        assert lib.fn[name](C.byref(b), None) == -1  # ({}: no results, no gradients)
    assert (lib.fn["block_workspace"](C.byref(b)) == -1) == bool(wrong)
    b = capi.Block(rows=4, width=16, eps=1e-6, x=64, block=64, post=64, res=64, pre=64, grad_x=64, grad_block=64, grad_post=64, grad_res=64, grad_pre=64, workspace=64, workspace_bytes=8)
    assert lib.fn["block_backward"](C.byref(b), None) == -1 and b"workspace" in lib.fn["last_error"]()


def test_clip_entries_refuse():
    lib = _lib.policy_binding()
    one = lambda t, x: (t * 1)(x)  # noqa: E731
    ptr, count, dtype = one(C.c_void_p, 64), one(C.c_int64, 100), one(C.c_int32, 0)
    call = lambda p=ptr, c=count, d=dtype, n=1, kind=2, most=1.0, norm=64, ws=64, size=1 << 20: lib.fn["clip"](p, c, d, n, kind, most, norm, ws, size, None)  # noqa: E731
    wrong = [dict(n=-1), dict(n=1 << 30), dict(c=None), dict(d=None), dict(p=None), dict(c=one(C.c_int64, -1)), dict(c=one(C.c_int64, 1 << 50)), dict(d=one(C.c_int32, 5)), dict(kind=1),
             dict(most=-1.0), dict(most=math.nan), dict(norm=None), dict(p=one(C.c_void_p, None)), dict(p=one(C.c_void_p, 66)), dict(ws=None), dict(size=0), dict(ws=68)]  # fmt: skip
    for kw in wrong:
        assert call(**kw) == -1, kw
    assert lib.fn["clip_workspace"](count, dtype, 1) == 8 and lib.fn["clip_workspace"](None, None, 0) == 0 and lib.fn["clip_workspace"](count, dtype, -3) == -1


# ---- refusals of the Python entries (fake tensors: shapes, types and devices without a GPU) ------------------------------------


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield lambda *shape, dtype=torch.float32, device="cuda", grad=False: torch.empty(*shape, dtype=dtype, device=device, requires_grad=grad)


def test_attention_refuses(fake):
    def call(q=None, k=None, v=None, g=None, **kw):
        pick = lambda x, *shape: fake(*shape) if x is None else x  # noqa: E731
        return ops.decay_attention(pick(q, 5, 3, 2, 16), pick(k, 5, 3, 2, 16), pick(v, 5, 3, 2, 8), pick(g, 2), **kw)

    bad = [
        (TypeError, dict(q=[1.0])), (ValueError, dict(q=fake(5, 3, 2, 16, device="cpu"))), (TypeError, dict(q=fake(5, 3, 2, 16, dtype=torch.float16))),
        (TypeError, dict(q=fake(5, 3, 2, 16, dtype=torch.float64))), (ValueError, dict(q=fake(3, 2, 16))), (ValueError, dict(k=fake(5, 3, 2, 17))), (ValueError, dict(k=fake(5, 3, 1, 16))),
        (TypeError, dict(k=fake(5, 3, 2, 16, dtype=torch.bfloat16))), (ValueError, dict(v=fake(5, 4, 2, 8))), (ValueError, dict(v=fake(5, 3, 2))), (ValueError, dict(v=fake(5, 3, 2, 129))),
        (ValueError, dict(v=fake(5, 3, 2, 0))), (ValueError, dict(g=fake(3))), (ValueError, dict(g=fake(2, grad=True))), (TypeError, dict(g=fake(2, dtype=torch.float64))),
        (ValueError, dict(g=fake(2, device="cpu"))), (ValueError, dict(initial_state=fake(3, 2, 8, 16))), (TypeError, dict(initial_state=fake(3, 2, 16, 8, dtype=torch.bfloat16))),
        (ValueError, dict(reset=fake(3, 5, dtype=torch.bool))), (TypeError, dict(reset=fake(5, 3, dtype=torch.int32))), (ValueError, dict(reset=fake(5, 3, dtype=torch.bool, device="cpu"))),
        (ValueError, dict(lengths=fake(5, dtype=torch.int32))), (TypeError, dict(lengths=fake(3, dtype=torch.int64))), (ValueError, dict(scale=math.nan)), (ValueError, dict(scale=math.inf)),
        (ValueError, dict(q=fake(5, 3, 0, 16), k=fake(5, 3, 0, 16), v=fake(5, 3, 0, 8), g=fake(0))), (ValueError, dict(q=fake(5, 3, 2, 130), k=fake(5, 3, 2, 130))),
    ]  # fmt: skip
    for error, kw in bad:
        with pytest.raises(error):
            call(**kw)


def test_step_refuses(fake):
    def call(q=None, state=None, **kw):
        pick = lambda x, *shape: fake(*shape) if x is None else x  # noqa: E731
        return ops.decay_attention_step(pick(q, 3, 2, 16), fake(3, 2, 16), fake(3, 2, 8), fake(2), pick(state, 3, 2, 16, 8), **kw)

    bad = [
        (ValueError, dict(q=fake(1, 3, 2, 16))), (ValueError, dict(state=fake(3, 2, 8, 16))), (ValueError, dict(state=fake(3, 2, 8, 16).transpose(2, 3))), (ValueError, dict(q=fake(3, 2, 16, grad=True))),
        (ValueError, dict(state=fake(3, 2, 16, 8, grad=True))), (ValueError, dict(reset=fake(2, dtype=torch.bool))), (TypeError, dict(skip=fake(3))), (ValueError, dict(skip=fake(3, 1, dtype=torch.uint8))),
        (TypeError, dict(state=fake(3, 2, 16, 8, dtype=torch.bfloat16))), (TypeError, dict(state=3)),
    ]  # fmt: skip
    for error, kw in bad:
        with pytest.raises(error):
            call(**kw)
    with pytest.raises(TypeError):
        ops.decay_attention_step(fake(3, 2, 16), fake(3, 2, 16), fake(3, 2, 8), fake(2), None)


def test_block_refuses(fake):
    def call(x=None, block=None, gate=None, post=None, res=None, pre=None, eps=1e-6):
        pick = lambda t, *shape: fake(*shape) if t is None else t  # noqa: E731
        return ops.gated_residual_norm(pick(x, 4, 16), pick(block, 4, 16), gate, pick(post, 16), pick(res, 16), pick(pre, 16), eps)

    bad = [
        (TypeError, dict(x=1.0)), (ValueError, dict(x=fake(4, 16, device="cpu"))), (TypeError, dict(x=fake(4, 16, dtype=torch.float16))), (ValueError, dict(block=fake(4, 15))),
        (ValueError, dict(gate=fake(1, 16))), (TypeError, dict(gate=fake(4, 16, dtype=torch.bfloat16))), (ValueError, dict(post=fake(1))), (TypeError, dict(res=fake(16, dtype=torch.bfloat16))),
        (TypeError, dict(res=0.5)), (ValueError, dict(pre=fake(16, device="cpu"))), (ValueError, dict(eps=0.0)), (ValueError, dict(eps=math.nan)), (ValueError, dict(x=fake(()))),
        (ValueError, dict(x=fake(4, 8193), block=fake(4, 8193), post=fake(8193), res=fake(8193), pre=fake(8193))), (ValueError, dict(x=fake(4, 0), block=fake(4, 0), post=fake(0), res=fake(0), pre=fake(0))),
    ]  # fmt: skip
    for error, kw in bad:
        with pytest.raises(error):
            call(**kw)


def test_clip_refuses(fake):
    g = fake(8)
    bad = [
        (ValueError, [fake(8, device="cpu")], {}), (TypeError, [fake(8, dtype=torch.float16)], {}), (TypeError, [g, 3.0], {}), (ValueError, [fake(8, grad=True)], {}), (ValueError, [g[::2]], {}),
        (ValueError, [fake(1).expand(8)], {}), (ValueError, [g], dict(max_norm=-1.0)), (ValueError, [g], dict(max_norm=math.nan)), (ValueError, [g], dict(norm_type=1.0)),
        (ValueError, [g], dict(norm_type=math.nan)), (ValueError, [fake(8).to_sparse()] if False else [fake(4, 4)[:, :3]], {}),
    ]  # fmt: skip
    for error, grads, kw in bad:
        with pytest.raises(error):
            ops.clip_grad_norm(grads, **{"max_norm": 1.0, **kw})
    assert float(ops.clip_grad_norm([None], 1.0).shape == ()) == 1.0


def test_dense_in_any_order():
    t = torch.zeros(3, 4, 5)
    assert all(ops._dense(x) for x in (t, t.permute(2, 0, 1), t.transpose(0, 1), t[1], t[:, :1, :][:1], torch.zeros(()), t[0:0]))
    assert not any(ops._dense(x) for x in (t[:, ::2], t[..., :2], t[:, :, :1].expand(3, 4, 5), t[:, 1:3]))


def test_clip_refuses_what_overlaps(monkeypatch):
    """the spans are compared on the host: told with CPU tensors that pass for the GPU's"""
    monkeypatch.setattr(ops, "_tensor", lambda *a, **k: None)
    t = torch.zeros(100)
    for grads in ([t, t], [t[:50], t[49:]], [t[10:20], t], [t[:60], torch.zeros(4), t[30:40]]):
        with pytest.raises(ValueError, match="share memory"):
            ops.clip_grad_norm(grads, 1.0)


# ---- the references ----------------------------------------------------------------------------------------------------------------


def test_reference_gradients_against_differences():
    gen = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    T, N, H, dk, dv = 9, 3, 2, 4, 5
    p = dict(q=rand(T, N, H, dk), k=rand(T, N, H, dk), v=rand(T, N, H, dv), log_decay=torch.tensor([-0.3, -0.01]), state=rand(N, H, dk, dv), scale=0.7)
    p["reset"] = torch.rand(T, N, generator=gen) < 0.2
    p["lengths"] = torch.tensor([T, 4, 0])
    dout, dlast = rand(T, N, H, dv), rand(N, H, dk, dv)
    d = ref.attention(**p, dout=dout, dlast=dlast)

    def value(p):
        r = ref.attention(**p)
        return (r["out"] * dout).sum() + (r["state"] * dlast).sum()

    for key in ("q", "k", "v", "state"):  # linear in each: the difference is exact
        e = rand(*p[key].shape)
        slope = (value({**p, key: p[key] + e}) - value({**p, key: p[key] - e})) / 2
        assert abs(slope - (d["d" + key] * e).sum()) < 1e-10
    args = [rand(4, 6), rand(4, 6), rand(4, 6), rand(6), rand(6), rand(6)]
    dy, dz = rand(4, 6), rand(4, 6)
    r = ref.block(*args, 1e-2, dy, dz)
    for i, key in enumerate(("dx", "dblock", "dgate", "dpost", "dres", "dpre")):
        e, h = rand(*args[i].shape), 1e-6
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * h * e
            o = ref.block(*moved, 1e-2)
            ends.append((o["y"] * dy).sum() + (o["z"] * dz).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - (r[key] * e).sum()) < 1e-7
