"""The policy operators' HIP kernels against plain 64-bit implementations (tests/policy_reference.py), at the sizes and masks where they can go wrong."""
import math

import pytest
import torch

import policy_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from rl4mm_amd import policy_ops

    return policy_ops


def normal(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def decays(H):
    return torch.log1p(-torch.exp2(-2.0 - torch.arange(H, dtype=torch.float64))).float().cuda()


def problem(seed, T, N, H, dk, dv, dtype, resets=0.0, ragged=False):
    gen = torch.Generator().manual_seed(seed + 1000)
    p = dict(q=normal(seed, T, N, H, dk, dtype=dtype), k=normal(seed + 1, T, N, H, dk, dtype=dtype), v=normal(seed + 2, T, N, H, dv, dtype=dtype), log_decay=decays(H))
    p["state"] = normal(seed + 3, N, H, dk, dv)
    p["reset"] = (torch.rand(T, N, generator=gen) < resets).cuda() if resets else None
    p["lengths"] = torch.randint(0, T + 1, (N,), generator=gen, dtype=torch.int32).cuda() if ragged else None
    p["scale"] = dk**-0.5
    return p, normal(seed + 4, T, N, H, dv, dtype=dtype), normal(seed + 5, N, H, dk, dv)


def run(ops, p, dout=None, dlast=None):
    """decay_attention, and its gradients where one of the outputs has one -> dict like the reference's"""
    kw = dict(reset=p["reset"], lengths=p["lengths"], scale=p["scale"])
    leaves = [x.detach().requires_grad_(True) for x in (p["q"], p["k"], p["v"], p["state"])]
    train = dout is not None or dlast is not None
    q, k, v, s = leaves if train else (x.detach() for x in leaves)
    out, last = ops.decay_attention(q, k, v, p["log_decay"], initial_state=s, **kw)
    got = {"out": out, "state": last}
    if train:
        pairs = [(o, d) for o, d in ((out, dout), (last, dlast)) if d is not None]
        grads = torch.autograd.grad([o for o, _ in pairs], leaves, [d for _, d in pairs])
        got.update(zip(("dq", "dk", "dv", "dstate"), grads))
    return got


def check(got, p, dout=None, dlast=None):
    want, tol = ref.attention(**p, dout=dout, dlast=dlast), ref.attention_tolerance(**p, dout=dout, dlast=dlast)
    for key, g in got.items():
        ref.close(g, want[key], tol[key], key)


# ---- decay attention over segments ----------------------------------------------------------------------------------------------

SIZES = [  # T, N, H, dk, dv
    (1, 1, 1, 1, 1), (1, 3, 2, 64, 64), (2, 2, 1, 16, 8), (15, 2, 3, 32, 32), (16, 1, 2, 17, 5), (17, 2, 2, 48, 80), (63, 2, 1, 64, 64), (64, 3, 2, 64, 64),
    (65, 1, 2, 64, 64), (100, 2, 1, 128, 128), (128, 1, 3, 100, 30), (130, 2, 2, 24, 128), (200, 2, 1, 33, 127), (333, 1, 2, 32, 64), (600, 1, 1, 64, 32),
]  # fmt: skip


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_attention_and_gradients(ops, size, dtype):
    p, dout, dlast = problem(11, *size, dtype)
    check(run(ops, p), p)
    check(run(ops, p, dout, dlast), p, dout, dlast)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("steps", [1, 17, 31, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("widths", [(128, 128), (128, 24), (30, 100), (64, 32), (12, 7)], ids=str)
def test_segments_about_a_chunk(ops, widths, steps, dtype):
    """Segments as long as a chunk, one token shorter and longer; then with numbers that are none behind the sequences' ends, which computes token by token"""
    p, dout, dlast = problem(steps + widths[1], steps, 5, 2, *widths, dtype, 0.1, True)
    check(run(ops, p, dout, dlast), p, dout, dlast)
    behind = torch.arange(steps, device="cuda")[:, None] >= p["lengths"][None]
    dirty = {**p, **{key: torch.where(behind[:, :, None, None], math.nan, p[key]) for key in ("q", "k", "v")}}
    check(run(ops, dirty, dout, dlast), p, dout, dlast)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(20, 9, 2, 32, 32), (64, 7, 1, 48, 80), (150, 6, 2, 64, 64), (257, 5, 1, 128, 128), (90, 5, 2, 7, 13), (30, 5, 2, 20, 50), (31, 5, 1, 50, 20), (32, 5, 1, 64, 64), (50, 4, 1, 5, 3), (28, 4, 1, 33, 64)], ids=str)
def test_resets_and_lengths(ops, size, dtype):
    for resets, ragged in ((0.05, False), (0.0, True), (0.02, True), (0.6, True)):
        p, dout, dlast = problem(int(100 * resets) + 3 * ragged, *size, dtype, resets, ragged)
        check(run(ops, p, dout, dlast), p, dout, dlast)


@pytest.mark.parametrize("at", [[0], [1], [15, 16], [63], [64], [65], [62, 63, 64, 65], [127, 128], list(range(130))], ids=lambda a: f"at{a[0]}x{len(a)}")
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_resets_at_the_borders(ops, at, dtype):
    p, dout, dlast = problem(5, 130, 2, 1, 32, 32, dtype)
    p["reset"] = torch.zeros(130, 2, dtype=torch.uint8, device="cuda")
    p["reset"][at, 1] = 1
    check(run(ops, p, dout, dlast), p, dout, dlast)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_lengths_at_the_borders(ops, dtype):
    lengths = [0, 1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 130, 131, -5, 2**31 - 1]
    p, dout, dlast = problem(6, 130, len(lengths), 1, 32, 48, dtype, resets=0.01)
    p["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = run(ops, p, dout, dlast)
    check(got, p, dout, dlast)
    assert torch.equal(got["state"][0], p["state"][0]) and torch.equal(got["dstate"][0], dlast[0])  # no token: they pass through


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("size", [(200, 4, 2, 64, 64), (200, 4, 1, 32, 128), (40, 4, 1, 30, 21), (30, 4, 2, 24, 60), (30, 4, 1, 60, 24), (30, 4, 1, 64, 64)], ids=str)
def test_masked_places_hold_anything(ops, size, junk, dtype):
    """Behind an environment's last token, before a reset, in the state that a reset drops: whatever is there reaches nothing else."""
    T = size[0]
    p, dout, dlast = problem(7, *size, dtype, resets=0.01)
    p["lengths"] = torch.tensor([T // 3, T, T, T], dtype=torch.int32, device="cuda")
    clean = {k: x.clone() for k, x in p.items() if isinstance(x, torch.Tensor)}
    cut = T // 2 + 1  # not at a tile's border
    p["reset"][cut, 1] = clean["reset"][cut, 1] = True
    p["reset"][0, 2] = clean["reset"][0, 2] = True
    for key in ("q", "k", "v"):
        p[key][T // 3:, 0] = junk  # behind the end
        p[key][cut - 3, 1] = junk  # an episode that went wrong, cut off
        clean[key][T // 3:, 0], clean[key][cut - 3, 1] = 0.0, 0.0
    p["state"][2] = junk
    clean["state"][2] = 0.0
    dirty = dout.clone()
    dirty[T // 3:, 0] = junk
    tidy = dout.clone()
    tidy[T // 3:, 0] = 0.0
    got = run(ops, p, dirty, dlast)
    q = {**p, **clean}
    want, tol = ref.attention(**q, dout=tidy, dlast=dlast), ref.attention_tolerance(**q, dout=tidy, dlast=dlast)
    for key, g in got.items():
        w, t = want[key], tol[key]
        if key in ("state", "dstate"):
            for n in (0, 1, 3) if key == "dstate" else (0, 1, 2, 3):
                if key == "dstate" and n == 1:
                    continue  # (the wrong episode's own gradient)
                ref.close(g[n], w[n], t[n], f"{key}[{n}]")
        else:
            for n in (0, 2, 3):
                ref.close(g[:, n], w[:, n], t[:, n], f"{key}[:, {n}]")
            ref.close(g[cut:, 1], w[cut:, 1], t[cut:, 1], f"{key}[cut:, 1]")
    # and the past does not see the future
    ref.close(got["out"][: cut - 3, 1], want["out"][: cut - 3, 1], tol["out"][: cut - 3, 1], "out before")
    assert not torch.isfinite(got["out"][cut - 3, 1].float()).any()


def test_future_gradients_do_not_reach_behind_a_reset(ops):
    """A gradient that is not a number stays in its episode, and does not reach later tokens of it."""
    p, dout, dlast = problem(8, 150, 2, 1, 32, 32, F32)
    p["reset"] = torch.zeros(150, 2, dtype=torch.bool, device="cuda")
    p["reset"][70] = True
    clean = dout.clone()
    dout[100, 0] = math.nan
    got, want, tol = run(ops, p, dout, dlast), ref.attention(**p, dout=clean, dlast=dlast), ref.attention_tolerance(**p, dout=clean, dlast=dlast)
    for key in ("dq", "dk", "dv"):
        ref.close(got[key][:, 1], want[key][:, 1], tol[key][:, 1], key)
        ref.close(got[key][:70, 0], want[key][:70, 0], tol[key][:70, 0], key)
        ref.close(got[key][101:, 0], want[key][101:, 0], tol[key][101:, 0], key)
    ref.close(got["dstate"], want["dstate"], tol["dstate"], "dstate")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides(ops, dtype):
    """views of one projection; environment-major storage; a stride of 0; an odd offset; a gradient that came through an expansion"""
    T, N, H, dk, dv = 70, 3, 2, 40, 24
    p, dout, dlast = problem(9, T, N, H, dk, dv, dtype, 0.02, True)
    both = torch.cat([p["q"].flatten(2), p["k"].flatten(2), p["v"].flatten(2)], -1)
    views = dict(zip("qkv", (x.unflatten(-1, (H, -1)) for x in both.split([H * dk, H * dk, H * dv], -1))))
    check(run(ops, {**p, **views}, dout, dlast), p, dout, dlast)
    major = {key: p[key].transpose(0, 1).contiguous().transpose(0, 1) for key in "qkv"}
    check(run(ops, {**p, **major}, dout.transpose(0, 2).contiguous().transpose(0, 2), dlast.transpose(2, 3).contiguous().transpose(2, 3)), p, dout, dlast)
    odd = {}
    for key in "qkv":
        room = torch.zeros(p[key].numel() + 1, dtype=dtype, device="cuda")
        odd[key] = room[1:].view(p[key].shape).copy_(p[key])
    check(run(ops, {**p, **odd}, dout, dlast), p, dout, dlast)
    last = {key: p[key].transpose(2, 3).contiguous().transpose(2, 3) for key in "qkv"}
    check(run(ops, {**p, **last}, dout, dlast), p, dout, dlast)
    one = {**p, "k": p["k"][:, :, :1].expand(T, N, H, dk), "v": p["v"][:1].expand(T, N, H, dv)}
    flat = {**one, "reset": one["reset"][:, :1].expand(T, N)}
    check(run(ops, flat, dout[:, :1].expand(T, N, H, dv), dlast), flat, dout[:, :1].expand(T, N, H, dv), dlast)
    # shared heads: the gradient of what was expanded is the sum over the heads
    shared = p["k"][:, :, :1].detach().requires_grad_(True)
    out, _ = ops.decay_attention(p["q"], shared.expand(T, N, H, dk), p["v"], p["log_decay"], initial_state=p["state"], reset=p["reset"], lengths=p["lengths"], scale=p["scale"])
    (dshared,) = torch.autograd.grad(out, shared, dout)
    full = {**p, "k": shared.detach().expand(T, N, H, dk)}
    want, tol = ref.attention(**full, dout=dout)["dk"].sum(2, keepdim=True), ref.attention_tolerance(**full, dout=dout)["dk"].sum(2, keepdim=True)
    ref.close(dshared, want, tol + 2 * ref.HALF[dtype] * want.abs(), "shared")


@pytest.mark.parametrize("size", [(70, 3, 2, 40, 24), (64, 2, 2, 64, 64)], ids=str)
def test_which_gradients_are_given_and_wanted(ops, size):
    p, dout, dlast = problem(10, *size, F32, 0.02)
    check(run(ops, p, dout, None), p, dout, None)
    check(run(ops, p, None, dlast), p, None, dlast)
    none = {**p, "state": None}
    q = p["q"].detach().requires_grad_(True)
    out, last = ops.decay_attention(q, p["k"], p["v"], p["log_decay"], reset=p["reset"], scale=p["scale"])
    (dq,) = torch.autograd.grad([out, last], [q], [dout, dlast])
    want, tol = ref.attention(**none, dout=dout, dlast=dlast), ref.attention_tolerance(**none, dout=dout, dlast=dlast)
    for key, g in (("out", out), ("state", last), ("dq", dq)):
        ref.close(g, want[key], tol[key], key)
    assert out.grad_fn is not None and not ops.decay_attention(q.detach(), p["k"], p["v"], p["log_decay"])[0].requires_grad
    with torch.no_grad():
        assert not ops.decay_attention(q, p["k"], p["v"], p["log_decay"])[0].requires_grad
    v = p["v"].detach().requires_grad_(True)  # the default scale
    out, _ = ops.decay_attention(p["q"], p["k"], v, p["log_decay"])
    ref.close(out, ref.attention(p["q"], p["k"], v, p["log_decay"], scale=size[3] ** -0.5)["out"], ref.attention_tolerance(p["q"], p["k"], v, p["log_decay"], scale=size[3] ** -0.5)["out"])


def test_gradients_against_differences(ops):
    """The output is linear in each operand: a difference over any step is exact but for rounding."""
    p, dout, dlast = problem(12, 90, 2, 2, 32, 48, F32, 0.02, True)
    got = run(ops, p, dout, dlast)

    def value(q):
        o = run(ops, q)
        return float((o["out"].double() * dout.double()).sum() + (o["state"].double() * dlast.double()).sum())

    tol = ref.attention_tolerance(**p)
    noise = 3 * float((tol["out"] * dout.double().cpu().abs()).sum() + (tol["state"] * dlast.double().cpu().abs()).sum())
    for key in ("q", "k", "v", "state"):
        d = normal(77, *p[key].shape)
        up, down = value({**p, key: p[key] + d}), value({**p, key: p[key] - d})
        assert abs((up - down) / 2 - float((got["d" + key].double() * d.double()).sum())) <= noise, key


@pytest.mark.parametrize("log_decay", [0.0, -1e-6, -30.0, -200.0, -math.inf, 0.01])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decays(ops, log_decay, dtype):
    p, dout, dlast = problem(13, 140, 2, 1, 32, 32, dtype, 0.01)
    p["log_decay"] = torch.tensor([log_decay], device="cuda")
    check(run(ops, p, dout, dlast), p, dout, dlast)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_a_long_axis(ops, dtype):
    """One environment, thousands of steps: the work is split over the steps."""
    p, dout, dlast = problem(14, 5000, 1, 2, 32, 32, dtype, 0.001)
    p["log_decay"] = torch.tensor([-1e-4, -0.02], device="cuda")
    check(run(ops, p, dout, dlast), p, dout, dlast)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(48, 80), (128, 64), (30, 21)], ids=str)
def test_a_long_axis_with_masks(ops, size, dtype):
    """lengths that end before, at and behind the borders of its parts; resets there; a part without one"""
    lengths = [0, 1, 255, 256, 257, 511, 512, 1000, 1023, 1024, 1100, 1099]
    p, dout, dlast = problem(15, 1100, len(lengths), 1, *size, dtype)
    p["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    p["reset"] = torch.zeros(1100, len(lengths), dtype=torch.bool, device="cuda")
    for t, n in ((256, 7), (255, 8), (512, 9), (513, 9), (1023, 10), (0, 10), (100, 6), (1098, 11), (1099, 11), (843, 11), (844, 10), (588, 11), (75, 10)):
        p["reset"][t, n] = True
    p["log_decay"] = torch.tensor([-0.002], device="cuda")
    check(run(ops, p, dout, dlast), p, dout, dlast)
    one = {**p, **{key: p[key][:, 3:4] for key in ("q", "k", "v", "reset")}, "state": p["state"][3:4], "lengths": None}
    check(run(ops, one, dout[:, 3:4], dlast[3:4]), one, dout[:, 3:4], dlast[3:4])


def test_empty(ops):
    for shape in ((0, 3, 2), (5, 0, 2)):
        q, v, s = torch.zeros(*shape, 8, device="cuda"), torch.zeros(*shape, 4, device="cuda", requires_grad=True), normal(1, shape[1], 2, 8, 4).requires_grad_(True)
        out, last = ops.decay_attention(q, q, v, decays(2), initial_state=s)
        assert out.shape == v.shape and torch.equal(last, s)
        torch.autograd.grad([out.sum() + last.sum()], [v, s])
    assert ops.decay_attention_step(q[0], q[0], v[0].detach(), decays(2), s.detach()).shape == (0, 2, 4)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(0, 3, 2), (5, 0, 2)], ids=str)
def test_empty_reaches_every_operand(ops, shape, dtype):
    """Each result of a segment without tokens has a gradient for each operand, like any other's: zeros, and the state's own."""
    leaves = [normal(k, *shape, d, dtype=dtype).requires_grad_(True) for k, d in enumerate((8, 8, 4))] + [normal(3, shape[1], 2, 8, 4).requires_grad_(True)]
    out, last = ops.decay_attention(*leaves[:3], decays(2), initial_state=leaves[3])
    assert out.dtype == dtype and out.shape == (*shape, 4) and torch.equal(last, leaves[3])
    for result, own in ((out, 0.0), (last, 1.0)):
        grads = torch.autograd.grad(result.sum(), leaves, retain_graph=True)
        assert all(g.shape == x.shape and g.dtype == x.dtype for g, x in zip(grads, leaves)) and torch.equal(grads[3], torch.full_like(grads[3], own))
    out, last = ops.decay_attention(*leaves[:3], decays(2))
    assert out.shape == (*shape, 4) and not last.any() and last.shape == (shape[1], 2, 8, 4)


# ---- one token of every environment ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (5, 2, 64, 64), (3, 3, 128, 128), (4, 1, 17, 5), (300, 2, 32, 32), (7, 2, 48, 80), (2, 2, 100, 31), (3, 1, 9, 100), (3, 2, 40, 3), (5, 1, 16, 4), (3, 2, 33, 127), (2, 1, 128, 33), (4, 2, 3, 7)], ids=str)
def test_step(ops, size, dtype):
    N, H, dk, dv = size
    p, _, _ = problem(20, 3, N, H, dk, dv, dtype)
    gen = torch.Generator().manual_seed(1)
    reset, skip = (torch.rand(3, N, generator=gen) < 0.3).cuda(), (torch.rand(3, N, generator=gen) < 0.3).cuda()
    state = p["state"].clone()
    for t in range(3):
        before = state.clone()
        out = ops.decay_attention_step(p["q"][t], p["k"][t], p["v"][t], p["log_decay"], state, reset=reset[t], skip=skip[t], scale=p["scale"])
        one = dict(q=p["q"][t:t + 1], k=p["k"][t:t + 1], v=p["v"][t:t + 1], log_decay=p["log_decay"], state=before, reset=reset[t:t + 1], lengths=(~skip[t]).int(), scale=p["scale"])
        check({"out": out[None], "state": state}, one)
        assert torch.equal(state[skip[t]], before[skip[t]])


def test_step_masks_hold_anything(ops):
    p, _, _ = problem(21, 1, 4, 2, 64, 64, F32)
    state = p["state"].clone()
    state[0], state[1] = math.nan, math.inf
    p["q"][0, 1], p["k"][0, 1], p["v"][0, 1] = math.nan, math.nan, math.nan
    out = ops.decay_attention_step(p["q"][0], p["k"][0], p["v"][0], p["log_decay"], state, reset=torch.tensor([1, 0, 0, 0], dtype=torch.uint8, device="cuda"),
                                   skip=torch.tensor([0, 7, 0, 0], dtype=torch.uint8, device="cuda"), scale=p["scale"])  # fmt: skip
    assert torch.isfinite(out).all() and torch.isinf(state[1]).all() and torch.isfinite(state[[0, 2, 3]]).all() and not out[1].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_steps_are_the_segment(ops, dtype):
    """An episode acted step by step and evaluated as a segment: the same outputs and state, within what each may be off."""
    p, _, _ = problem(22, 75, 6, 2, 64, 64, dtype, 0.03)
    whole, tol = run(ops, p), ref.attention_tolerance(**p)
    state, outs = p["state"].clone(), []
    for t in range(75):
        outs.append(ops.decay_attention_step(p["q"][t], p["k"][t], p["v"][t], p["log_decay"], state, reset=p["reset"][t], scale=p["scale"]))
    ref.close(torch.stack(outs), whole["out"].double().cpu(), 2 * tol["out"], "out")
    ref.close(state, whole["state"].double().cpu(), 2 * tol["state"], "state")


def test_step_strides_and_modes(ops):
    p, _, _ = problem(23, 2, 5, 2, 48, 64, BF16)
    both = torch.cat([p["q"].flatten(2), p["k"].flatten(2), p["v"].flatten(2)], -1)[1]
    q, k, v = (x.unflatten(-1, (2, -1)) for x in both.split([96, 96, 128], -1))
    flags = torch.tensor([0, 1, 0, 0, 1, 0, 0, 0, 1, 0], dtype=torch.uint8, device="cuda")[::2]
    a, b = p["state"].clone(), p["state"].clone()
    one = ops.decay_attention_step(q, k, v, p["log_decay"], a, reset=flags, skip=flags.flip(0))
    two = ops.decay_attention_step(p["q"][1], p["k"][1], p["v"][1], p["log_decay"], b, reset=flags.contiguous(), skip=flags.flip(0).contiguous())
    assert torch.equal(one, two) and torch.equal(a, b)
    version = a._version
    with torch.inference_mode():
        ops.decay_attention_step(q, k, v, p["log_decay"], torch.zeros_like(a))
        ops.decay_attention_step(q, k, v, p["log_decay"], a)
    assert a._version > version
    leaf = torch.zeros_like(a).requires_grad_(True)
    x = p["q"][:1].float().requires_grad_(True)
    out, _ = ops.decay_attention(x, p["k"][:1].float(), p["v"][:1].float(), p["log_decay"], initial_state=leaf.detach())
    with pytest.raises(ValueError):
        ops.decay_attention_step(p["q"][0], p["k"][0], p["v"][0], p["log_decay"], leaf)


# ---- the block's end -------------------------------------------------------------------------------------------------------------


def block_problem(seed, rows, width, stream, dtype):
    shape = (rows, width)
    args = [normal(seed, *shape, dtype=stream), normal(seed + 1, *shape, dtype=dtype), normal(seed + 2, *shape, dtype=dtype)]
    args += [1 + 0.2 * normal(seed + 3, width), 0.5 * normal(seed + 4, width), 1 + 0.2 * normal(seed + 5, width)]
    return args, normal(seed + 6, *shape, dtype=stream), normal(seed + 7, *shape, dtype=dtype)


BLOCK_KEYS = ("dx", "dblock", "dgate", "dpost", "dres", "dpre")


def check_block(ops, args, dy, dz, eps=1e-6):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in args]
    y, z = ops.gated_residual_norm(*leaves, eps=eps)
    want, tol = ref.block(*args, eps, dy, dz), ref.block_tolerance(*args, eps, dy, dz)
    ref.close(y, want["y"], tol["y"], "y")
    ref.close(z, want["z"], tol["z"], "z")
    assert y.dtype == args[0].dtype and z.dtype == args[1].dtype
    pairs = [(o, d) for o, d in ((y, dy), (z, dz)) if d is not None]
    if pairs:
        grads = torch.autograd.grad([o for o, _ in pairs], [t for t in leaves if t is not None], [d for _, d in pairs])
        for key, g in zip([k for k, t in zip(BLOCK_KEYS, leaves) if t is not None], grads):
            ref.close(g, want[key], tol[key], key)
        return [y, z, *grads]
    return [y, z]


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)], ids=["f32", "bf16", "f32+bf16", "bf16+f32"])
@pytest.mark.parametrize("width", [1, 3, 4, 30, 64, 255, 256, 257, 264, 500, 512, 520, 1000, 1024, 1025, 1032, 2048, 2052, 5000, 8192])
def test_block(ops, width, types):
    for rows in (1, 7):
        args, dy, dz = block_problem(width, rows, width, *types)
        check_block(ops, args, dy, dz)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)], ids=["f32", "bf16", "f32+bf16", "bf16+f32"])
@pytest.mark.parametrize("width", [2049, 2056, 4088, 4094, 4096, 4097, 4104, 8191])
def test_block_wide_rows(ops, width, types):
    """each number of threads that shares a long row, full and a little more than full"""
    args, dy, dz = block_problem(width, 3, width, *types)
    check_block(ops, args, dy, dz)


def test_block_many_rows_and_order(ops):
    """More rows than workgroups: the weights' gradients, and twice the same bits"""
    for rows, width in ((5000, 32), (2500, 300), (1200, 1100)):
        args, dy, dz = block_problem(3, rows, width, BF16, BF16)
        a, b = check_block(ops, args, dy, dz), check_block(ops, args, dy, dz)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_block_parts(ops):
    """no gate; one gradient only; large and tiny values; zeros; another eps"""
    for width in (48, 1500):
        args, dy, dz = block_problem(5, 9, width, F32, F32)
        check_block(ops, [*args[:2], None, *args[3:]], dy, dz)
        check_block(ops, args, dy, None)
        check_block(ops, args, None, dz)
        check_block(ops, args, None, None)
        check_block(ops, args, dy, dz, eps=1e-3)
        check_block(ops, [args[0], args[1] * 0.0, *args[2:]], dy, dz)
        check_block(ops, [args[0], args[1] * 1e4, args[2] * 30.0, *args[3:]], dy, dz)


def test_block_strides(ops):
    args, dy, dz = block_problem(6, 24, 64, BF16, BF16)
    wide = torch.cat(args[:3], 1)
    cut = [wide[:, i * 64:(i + 1) * 64] for i in range(3)]
    plain = check_block(ops, args, dy, dz)
    strided = check_block(ops, [*cut, *args[3:]], torch.cat([dy, dy], 1)[:, 64:], dz.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(plain, strided))
    off = torch.zeros(24 * 64 + 1, dtype=BF16, device="cuda")[1:].view(24, 64).copy_(args[0])
    check_block(ops, [off, *args[1:]], dy, dz)
    three = [t.view(2, 12, 64) for t in args[:3]]
    y, z = ops.gated_residual_norm(*three, *args[3:])
    assert torch.equal(y.view(24, 64), plain[0]) and torch.equal(z.view(24, 64), plain[1])
    major = [t.view(2, 12, 64).transpose(0, 1) for t in args[:3]]  # rows in another order: strides that no single row stride describes
    y, z = ops.gated_residual_norm(*major, *args[3:])
    assert torch.equal(y.transpose(0, 1).reshape(24, 64), plain[0]) and torch.equal(z.transpose(0, 1).reshape(24, 64), plain[1])
    row = ops.gated_residual_norm(args[0][0], args[1][0], args[2][0], *args[3:])
    assert torch.equal(row[0], plain[0][0]) and torch.equal(row[1], plain[1][0])
    x, post = args[0].expand(24, 64), args[3]
    y, _ = ops.gated_residual_norm(args[0][:1].expand(24, 64), *args[1:])
    assert y.shape == (24, 64)
    post = torch.ones(64, device="cuda", requires_grad=True)
    y, z = ops.gated_residual_norm(args[0][:0], args[1][:0], args[2][:0], post, args[4], args[5])
    assert y.shape == z.shape == (0, 64) and not torch.autograd.grad(y.sum() + z.sum(), post)[0].any()


def test_block_gradients_against_differences(ops):
    args, dy, dz = block_problem(8, 5, 20, F32, F32)
    leaves = [t.detach().requires_grad_(True) for t in args]
    y, z = ops.gated_residual_norm(*leaves, eps=1e-2)
    grads = torch.autograd.grad([y, z], leaves, [dy, dz])

    def value(args):  # the plain form in 64 bits
        r = ref.block(*args, 1e-2)
        return float((r["y"] * dy.double().cpu()).sum() + (r["z"] * dz.double().cpu()).sum())

    for i, g in enumerate(grads):
        d = normal(90 + i, *args[i].shape).double().cpu()
        step = 1e-5  # error of the difference: about step^2 * third derivative + 2^-53 / step, both under 1e-9 of values of order 10
        wide = [t.double().cpu() for t in args]
        up, down = list(wide), list(wide)
        up[i], down[i] = wide[i] + step * d, wide[i] - step * d
        slope, mine = (value(up) - value(down)) / (2 * step), float((g.double().cpu() * d).sum())
        assert abs(slope - mine) <= 1e-5 * float((g.double().cpu() * d).abs().sum()) + 1e-7


# ---- the global norm -------------------------------------------------------------------------------------------------------------


def check_clip(ops, grads, max_norm, kind=2.0):
    """The norm within its type's rounding; every element within that of the factor, of the product and of its own type."""
    before = [g.clone() for g in grads]
    flat = torch.cat([g.double().reshape(-1) for g in grads]) if grads else torch.zeros(1)
    want = float(flat.square().sum().sqrt() if kind == 2.0 else flat.abs().max())
    norm = ops.clip_grad_norm(grads, max_norm, kind)
    assert norm.dtype == F32 and norm.shape == () and abs(float(norm) - want) <= 2**-23 * want
    by = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        if by == 1.0:
            assert torch.equal(g, b)
        else:
            w = b.double().cpu() * by
            ref.close(g, w, w.abs() * (2 * 2.0**-24 + ref.HALF[g.dtype] * (1 + 2.0**-22)) + (1e-45 if g.dtype == F32 else 1e-40), "gradient")


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0, math.inf])
def test_clip(ops, max_norm, kind):
    sizes = [1, 0, 3, 8, 255, 4096, 8191, 8192, 8193, 8200, 70001, 2]
    for types in ([F32], [BF16], [F32, BF16, BF16]):
        check_clip(ops, [normal(i, s, dtype=types[i % len(types)]) for i, s in enumerate(sizes)], max_norm, kind)


def test_clip_views_and_orders(ops):
    """Views at every offset, transposed tensors, matrices, scalars, a flat bucket cut into neighbours"""
    for dtype in (F32, BF16):
        bucket = normal(4, 100_000, dtype=dtype)
        cuts = [bucket[i * 9001 + i: (i + 1) * 9001 - i % 3] for i in range(11)]
        rest = bucket[99_050:].clone()
        check_clip(ops, cuts, 0.1)
        assert torch.equal(bucket[99_050:], rest)
        guard = normal(5, 2000, dtype=dtype)
        for offset in range(9):
            for size in (0, 1, 2, 7, 9, 63):
                around = guard.clone()
                check_clip(ops, [around[offset: offset + size]] if size else [around[:1]], 0.01)
                if size:
                    assert torch.equal(around[offset + size:], guard[offset + size:]) and torch.equal(around[:offset], guard[:offset])
        check_clip(ops, [normal(6, 30, 50, dtype=dtype).t(), normal(7, 3, 4, 5, dtype=dtype).permute(2, 0, 1), normal(8, dtype=dtype), normal(9, 4, 1, 6, dtype=dtype)], 0.1)


def test_clip_many_tensors(ops):
    check_clip(ops, [normal(i, 50 + 13 * (i % 40), dtype=(F32, BF16)[i % 2]) for i in range(700)], 1.0)
    check_clip(ops, [normal(1, 20_000_000), normal(2, 7_000_001, dtype=BF16)], 1.0)


def test_clip_extremes(ops):
    for dtype in (F32, BF16):
        check_clip(ops, [torch.full((1000,), 1e30, device="cuda", dtype=dtype)], 1.0)  # squares beyond 32 bits
        check_clip(ops, [torch.full((1000,), 1e-30, device="cuda", dtype=dtype)], 1e-31)
        for junk in (math.nan, math.inf):
            for kind in (2.0, math.inf):
                grads = [normal(1, 1000, dtype=dtype), normal(2, 500, dtype=dtype)]
                grads[1][77] = junk
                norm = ops.clip_grad_norm(grads, 1.0, kind)
                if math.isnan(junk):
                    assert torch.isnan(norm) and all(torch.isnan(g).all() for g in grads)
                else:
                    assert torch.isinf(norm) and not grads[0].any() and torch.isnan(grads[1][77]) and not grads[1][:77].any() and not grads[1][78:].any()


def test_clip_of_nothing_and_of_one(ops):
    assert float(ops.clip_grad_norm([], 1.0)) == 0.0 and float(ops.clip_grad_norm([None], 1.0)) == 0.0
    assert float(ops.clip_grad_norm(torch.zeros(0, device="cuda"), 1.0)) == 0.0
    g = normal(1, 3000)
    want = (g / g.double().norm().float()).clone()
    ops.clip_grad_norm((x for x in (None, g)), 1.0)
    assert torch.allclose(g, want, rtol=1e-5)
    with torch.inference_mode():
        ops.clip_grad_norm(torch.ones(5, device="cuda"), 1.0)


# ---- streams and graphs ----------------------------------------------------------------------------------------------------------


def everything(ops, p, dout, dlast, args, dy, dz, grads, state):
    """a pass through all of them -> their results, none of them the operands' own memory"""
    got = run(ops, p, dout, dlast)
    leaves = [t.detach().requires_grad_(True) for t in args]
    y, z = ops.gated_residual_norm(*leaves)
    more = torch.autograd.grad([y, z], leaves, [dy, dz])
    copies = [g.clone() for g in grads]
    norm = ops.clip_grad_norm(copies, 0.5)
    held = state.clone()
    step = ops.decay_attention_step(p["q"][0], p["k"][0], p["v"][0], p["log_decay"], held, reset=p["reset"][0])
    return [x.detach() for x in (*got.values(), y, z, *more, norm, *copies, step, held)]


def make_everything(seed):
    p, dout, dlast = problem(seed, 700, 2, 2, 64, 48, BF16, 0.01, True)
    args, dy, dz = block_problem(seed, 700, 260, F32, BF16)
    return p, dout, dlast, args, dy, dz, [normal(seed, 30_000), normal(seed + 1, 999, dtype=BF16)], p["state"]


def test_captured_and_replayed(ops):
    """One graph of all of them, its inputs changed in place: every replay is the eager result, with eager work between the replays."""
    inputs, fresh = make_everything(31), make_everything(57)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        everything(ops, *inputs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        results = everything(ops, *inputs)

    def flat(x):
        return [x] if isinstance(x, torch.Tensor) else [t for y in (x.values() if isinstance(x, dict) else x) for t in flat(y)] if isinstance(x, (list, tuple, dict)) else []

    for i in range(4):
        for a, b in zip(flat(list(inputs)), flat(list(fresh))):
            if a.is_floating_point() and a.dim() > 1 and i:
                a.mul_(0.5).add_(b, alpha=0.1 * i)
        graph.replay()
        torch.cuda.synchronize()
        want = everything(ops, *inputs)
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(results, want)):
            assert torch.equal(a, b), (i, n)


def test_two_streams_at_once(ops):
    one, two = make_everything(41), make_everything(43)
    want = [everything(ops, *one), everything(ops, *two)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for i, inputs in enumerate((one, two)):
            with torch.cuda.stream(streams[i]):
                got[i] = everything(ops, *inputs)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_two_threads_at_once(ops):
    import threading

    sides = [make_everything(41), make_everything(43)]
    want = [everything(ops, *s) for s in sides]
    torch.cuda.synchronize()
    got, wrong = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(3):
                    got[i] = everything(ops, *sides[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not wrong
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


# ---- beyond 32 bits of elements and offsets ----------------------------------------------------------------------------------------


def test_attention_beyond_32_bits(ops):
    """The last environments of a batch of more than 2^31 elements are what they are alone: each environment's arithmetic is its own."""
    N = 131_100
    x = torch.randn(64, N, 4, 64, device="cuda", dtype=BF16)
    assert x.numel() > 2**31
    g, reset = decays(4), torch.zeros(64, N, dtype=torch.bool, device="cuda")
    reset[17, -2:] = True
    leaf = x.requires_grad_(True)
    out, last = ops.decay_attention(leaf, leaf.detach(), leaf.detach(), g, reset=reset)
    (dx,) = torch.autograd.grad(out, leaf, x.detach())
    alone = x.detach()[:, -2:].contiguous().requires_grad_(True)
    out2, last2 = ops.decay_attention(alone, alone.detach(), alone.detach(), g, reset=reset[:, -2:].contiguous())
    (dx2,) = torch.autograd.grad(out2, alone, alone.detach())
    assert torch.equal(out[:, -2:], out2) and torch.equal(last[-2:], last2) and torch.equal(dx[:, -2:], dx2)
    state = last.detach()
    now = x.detach()[5]
    tail = state[-2:].clone()
    one = ops.decay_attention_step(now, now, now, g, state)
    two = ops.decay_attention_step(now[-2:], now[-2:], now[-2:], g, tail)
    assert torch.equal(one[-2:], two) and torch.equal(state[-2:], tail)


def test_block_and_clip_beyond_32_bits(ops):
    x = torch.randn(8_388_700, 256, device="cuda", dtype=BF16)
    assert x.numel() > 2**31
    w = [1 + 0.1 * normal(i, 256) for i in range(3)]
    leaf = x.requires_grad_(True)
    y, z = ops.gated_residual_norm(leaf, x.detach(), x.detach(), *w)
    (dx,) = torch.autograd.grad([y, z], leaf, [x.detach(), x.detach()])
    alone = x.detach()[-3:].clone().requires_grad_(True)
    y2, z2 = ops.gated_residual_norm(alone, alone.detach(), alone.detach(), *w)
    (dx2,) = torch.autograd.grad([y2, z2], alone, [alone.detach(), alone.detach()])
    assert torch.equal(y[-3:], y2) and torch.equal(z[-3:], z2) and torch.equal(dx[-3:], dx2)
    grad = x.detach()
    before = grad[-2:].clone()
    norm = ops.clip_grad_norm(grad, 1.0)
    assert abs(float(norm) / grad.numel() ** 0.5 - 1.0) < 0.01
    by = torch.tensor(1.0 / (float(norm) + 1e-6))
    assert torch.allclose(grad[-2:].float(), before.float() * by.cuda(), rtol=2.0**-7, atol=0.0)
