"""The policy operators' measured cases: what a policy that remembers order flow runs per environment step and per update.

kind "act"       decay_attention_step: one observation of every environment, the state of each updated in place
kind "sequence"  decay_attention over a recorded segment [T, N], alone or with its gradients ("train")
kind "clip"      clip_grad_norm over the gradients of all parameters
kind "block"     gated_residual_norm at the end of a block, alone or with its gradients

`run` computes them in plain torch, or (`own`) through rl4mm_amd.policy_ops."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
CHUNK = 64  # tokens that the plain form of "sequence" takes at a time


def _case(name, **kw):
    return dict(kw, name=name)


def listed():
    return [
        # a handful of evaluation environments, one step: latency
        _case("act_small", kind="act", envs=64, heads=4, dk=64, dv=64, dtype="f32"),
        # the benchmark's 4096 environments, one step
        _case("act_batch", kind="act", envs=4096, heads=8, dk=64, dv=64, dtype="bf16"),
        # a rollout segment evaluated without gradients (values for the advantages)
        _case("segment", kind="sequence", steps=128, envs=512, heads=4, dk=64, dv=64, dtype="bf16", train=False, ragged=False),
        # two whole 30-minute episodes at 0.1 s steps: few rows, a long axis
        _case("episode", kind="sequence", steps=18000, envs=2, heads=4, dk=64, dv=64, dtype="f32", train=False, ragged=False),
        # an update on 20-step segments of 4096 environments
        _case("update_short", kind="sequence", steps=20, envs=4096, heads=4, dk=32, dv=32, dtype="f32", train=True, ragged=False),
        # an update on long segments, some environments stopped early
        _case("update_long", kind="sequence", steps=4500, envs=16, heads=8, dk=128, dv=128, dtype="bf16", train=True, ragged=True),
        # nothing round: 37 environments, 333 steps, 3 heads of 48 and 80
        _case("update_odd", kind="sequence", steps=333, envs=37, heads=3, dk=48, dv=80, dtype="bf16", train=True, ragged=True),
        # the 2 x 256 policy's six tensors
        _case("clip_policy", kind="clip", tensors=6, values=69636, dtype="f32"),
        # a large model's gradients, two types among them
        _case("clip_large", kind="clip", tensors=60, values=150_000_000, dtype="mixed"),
        # the block's end for one step of 64 environments
        _case("block_act", kind="block", rows=64, width=256, stream="f32", dtype="f32", train=False),
        # the same in an update: 512 environments x 128 steps
        _case("block_update", kind="block", rows=65536, width=1024, stream="bf16", dtype="bf16", train=True),
        # an odd width, the residual stream in 32 bits
        _case("block_odd", kind="block", rows=4099, width=500, stream="f32", dtype="bf16", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["act", "sequence", "sequence", "clip", "block"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "act":
        heads, dk, dv = rng.randint(1, 8), rng.randint(8, 128), rng.randint(8, 128)
        envs = _log(rng, 1, max(2, min(16384, 134_000_000 // (heads * dk * dv))))
        return dict(kind=kind, envs=envs, heads=heads, dk=dk, dv=dv, dtype=dtype)
    if kind == "sequence":
        heads, dk, dv = rng.randint(1, 8), rng.randint(8, 128), rng.randint(8, 128)
        steps = _log(rng, 1, 18000)
        most = 60_000_000 // (heads * (dk + dv))
        envs = _log(rng, 1, max(2, min(4096, most // steps)))
        return dict(kind=kind, steps=steps, envs=envs, heads=heads, dk=dk, dv=dv, dtype=dtype, train=rng.random() < 0.6, ragged=rng.random() < 0.5)
    if kind == "clip":
        return dict(kind=kind, tensors=rng.randint(1, 60), values=_log(rng, 1000, 120_000_000), dtype=rng.choice(["f32", "bf16", "mixed"]))
    width = _log(rng, 8, 4096)
    return dict(kind=kind, rows=_log(rng, 1, max(2, 60_000_000 // width)), width=width, stream=rng.choice(["f32", dtype]), dtype=dtype, train=rng.random() < 0.6)


def _sizes(case):
    """The tensors' lengths: matrices and their biases, spread over a factor of a hundred, `values` in all."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["values"])
    share = [math.exp(rng.uniform(0.0, math.log(100.0))) * (1.0 if i % 2 == 0 else 0.004) for i in range(case["tensors"])]
    sizes = [max(1, int(case["values"] * s / sum(share))) for s in share]
    sizes[0] += max(0, case["values"] - sum(sizes))
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    def chance(p, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") < p

    s = dict(case)
    if case["kind"] in ("act", "sequence"):
        n, h, dk, dv, dtype = case["envs"], case["heads"], case["dk"], case["dv"], DTYPES[case["dtype"]]
        lead = (n,) if case["kind"] == "act" else (case["steps"], n)
        qkv = normal(*lead, h * (2 * dk + dv), dtype=dtype)  # one projection's output: the operands are views of it
        parts = qkv.split([h * dk, h * dk, h * dv], dim=-1)
        s["q"], s["k"], s["v"] = (p.unflatten(-1, (h, -1)) for p in parts)
        # memories of 16 steps and more, twice as long from head to head
        s["log_decay"] = torch.log1p(-torch.exp2(-4.0 - torch.arange(h, device="cuda", dtype=torch.float64))).float()
        s["scale"] = dk ** -0.5
        s["state"] = normal(n, h, dk, dv)
        s["reset"] = chance(0.005, *lead)  # an episode begins
        if case["kind"] == "act":
            s["skip"] = chance(0.02, n)  # environments that are done and sit out
        else:
            s["lengths"] = None
            if case["ragged"]:
                short = torch.randint(0, case["steps"] + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
                s["lengths"] = torch.where(chance(0.3, n), short, torch.full_like(short, case["steps"]))
            if case["train"]:
                s["dout"] = normal(*lead, h, dv, dtype=dtype)
                s["dstate"] = normal(n, h, dk, dv)
                for key in ("q", "k", "v", "state"):
                    s[key] = s[key].detach().requires_grad_(True)
    elif case["kind"] == "clip":
        kinds = [torch.float32, torch.bfloat16] if case["dtype"] == "mixed" else [DTYPES[case["dtype"]]]
        s["grads"] = [normal(m, dtype=kinds[(i // 2) % len(kinds)]).mul_(0.02) for i, m in enumerate(_sizes(case))]
        s["max_norm"] = 0.5  # annealed a little from pass to pass, so that each one clips
    else:
        rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
        s["x"], s["block"], s["gate"] = normal(rows, width, dtype=DTYPES[case["stream"]]), normal(rows, width, dtype=dtype), normal(rows, width, dtype=dtype)
        s["post"], s["pre"] = 1.0 + 0.1 * normal(width), 1.0 + 0.1 * normal(width)
        s["res"] = 0.3 + 0.05 * normal(width)
        if case["train"]:
            s["dy"], s["dz"] = normal(rows, width, dtype=DTYPES[case["stream"]]), normal(rows, width, dtype=dtype)
            for key in ("x", "block", "gate", "post", "pre", "res"):
                s[key].requires_grad_(True)
    return s


def run(s):
    if s["kind"] == "act":
        return _act(s)
    if s["kind"] == "sequence":
        return _sequence(s)
    if s["kind"] == "clip":
        return _clip(s)
    return _block(s)


def _act(s):
    if own:
        from rl4mm_amd import policy_ops

        out = policy_ops.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], reset=s["reset"], skip=s["skip"], scale=s["scale"])
        return {"out": out, "state": s["state"]}
    q, k, v, state = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    gone, kept = s["reset"][:, None, None, None], s["skip"][:, None, None, None]
    new = torch.where(gone, torch.zeros_like(state), state) * torch.exp(s["log_decay"])[:, None, None] + k[..., :, None] * v[..., None, :]
    out = (q[..., None, :] @ new).squeeze(-2) * s["scale"]
    state.copy_(torch.where(kept, state, new))
    return {"out": torch.where(kept[..., 0], torch.zeros_like(out), out).to(s["q"].dtype), "state": state}


def _plain_sequence(q, k, v, log_decay, state, reset, lengths, scale):
    """32-bit torch, a chunk at a time for the tokens of one chunk, a matrix over the chunks for what goes from one to the next."""
    t, n, h, dk = q.shape
    dv = v.shape[-1]
    c = min(CHUNK, t)
    m = -(-t // c)
    fill = m * c - t
    there = torch.arange(t, device=q.device)[:, None] < (lengths[None, :] if lengths is not None else t)  # [t, n] or [t, 1]
    there = there.expand(t, n)

    def chunks(x, value=0.0):  # [t, n, h, d] -> [n, h, m, c, d]
        x = torch.nn.functional.pad(x.movedim(0, 2), (0, 0, 0, fill), value=value)
        return x.unflatten(2, (m, c))

    keep = there[..., None, None]
    q, k, v = (chunks(torch.where(keep, x, torch.zeros_like(x))) for x in (q, k, v))
    # a token behind an environment's last one neither decays nor resets: its "time" stands still
    there = torch.nn.functional.pad(there, (0, 0, 0, fill))
    reset = torch.nn.functional.pad(reset, (0, 0, 0, fill)) & there
    time = there.double().cumsum(0).T.reshape(n, 1, m, c)  # tokens up to and with this one
    part = reset.double().cumsum(0).T.reshape(n, 1, m, c)  # resets up to and with it

    def decay(a, b, same):  # e^(g (a - b)) where `same`, else 0, its exponent in 64 bits: [n, 1, ...] -> [n, h, ...]
        gap = torch.where(same, a - b, torch.zeros_like(a - b))
        e = torch.exp(log_decay.double().reshape(-1, *[1] * (gap.dim() - 2)) * gap)
        return torch.where(same, e, torch.zeros_like(e)).float()

    tail_time, tail_part = time[..., -1:], part[..., -1:]
    head_time = torch.cat([torch.zeros_like(tail_time[:, :, :1]), tail_time[:, :, :-1]], 2)  # tokens before the chunk
    head_part = torch.cat([torch.zeros_like(tail_part[:, :, :1]), tail_part[:, :, :-1]], 2)
    order = torch.ones(c, c, dtype=torch.bool, device=q.device).tril()
    within = decay(time[..., :, None], time[..., None, :], order & (part[..., :, None] == part[..., None, :]))
    scores = (q @ k.transpose(-1, -2)) * within
    to_tail = decay(tail_time, time, part == tail_part)
    local = (k * to_tail[..., None]).transpose(-1, -2) @ v  # what each chunk adds to the state
    # the state after chunk i: what chunk j <= i added, and what was there at the start
    a, b = tail_time[..., 0][..., :, None], tail_time[..., 0][..., None, :]
    pa, pb = tail_part[..., 0][..., :, None], tail_part[..., 0][..., None, :]
    across = decay(a, b, torch.ones(m, m, dtype=torch.bool, device=q.device).tril() & (pa == pb))
    first = decay(tail_time[..., 0], torch.zeros_like(tail_time[..., 0]), tail_part[..., 0] == 0)
    after = (across @ local.flatten(-2)) + first[..., None] * state.flatten(-2)[:, :, None, :]
    before = torch.cat([state.flatten(-2)[:, :, None, :], after[:, :, :-1]], 2).unflatten(-1, (dk, dv))
    from_head = decay(time, head_time, part == head_part)
    out = (scores @ v + (q * from_head[..., None]) @ before) * scale
    out = out.flatten(2, 3)[:, :, :t].movedim(2, 0)
    return torch.where(keep, out, torch.zeros_like(out)), after[:, :, -1].unflatten(-1, (dk, dv))


def _sequence(s):
    keys = ("q", "k", "v", "state")
    if own:
        from rl4mm_amd import policy_ops

        out, last = policy_ops.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["state"], reset=s["reset"], lengths=s["lengths"], scale=s["scale"])
        got = {"out": out, "state": last}
        if s["train"]:
            grads = torch.autograd.grad([out, last], [s[key] for key in keys], [s["dout"], s["dstate"]])
            got = {"out": out.detach(), "state": last.detach(), **{"d" + key: d for key, d in zip(keys, grads)}}
        return got
    wide = [s[key].detach().float().requires_grad_(s["train"]) for key in keys]
    out, last = _plain_sequence(*wide[:3], s["log_decay"], wide[3], s["reset"], s["lengths"], s["scale"])
    got = {"out": out.detach().to(s["q"].dtype), "state": last.detach()}
    if s["train"]:
        grads = torch.autograd.grad([out, last], wide, [s["dout"].float(), s["dstate"]])
        got.update({"d" + key: d.to(s[key].dtype) for key, d in zip(keys, grads)})
    return got


def _clip(s):
    grads, most = s["grads"], s["max_norm"]
    s["max_norm"] = most * 0.9998
    if own:
        from rl4mm_amd import policy_ops

        norm = policy_ops.clip_grad_norm(grads, most)
    else:
        norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()
        by = torch.clamp(most / (norm + EPS), max=1.0).float()
        [g.copy_(g.float() * by) for g in grads]
        norm = norm.float()
    return [norm] + grads


def _block(s):
    keys = ("x", "block", "gate", "post", "res", "pre")
    if own:
        from rl4mm_amd import policy_ops

        y, z = policy_ops.gated_residual_norm(*(s[key] for key in keys), eps=EPS)
        got = {"y": y, "z": z}
        if s["train"]:
            grads = torch.autograd.grad([y, z], [s[key] for key in keys], [s["dy"], s["dz"]])
            got = {"y": y.detach(), "z": z.detach(), **{"d" + key: d for key, d in zip(keys, grads)}}
        return got
    wide = [s[key].detach().float().requires_grad_(s["train"]) for key in keys]
    x, block, gate, post, res, pre = wide
    normed = block * torch.rsqrt(block.square().mean(-1, keepdim=True) + EPS) * post
    y = x + res * normed / (1.0 + torch.exp(-gate))
    z = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * pre
    got = {"y": y.detach().to(s["x"].dtype), "z": z.detach().to(s["block"].dtype)}
    if s["train"]:
        grads = torch.autograd.grad([y, z], wide, [s["dy"].float(), s["dz"].float()])
        got.update({"d" + key: d.to(s[key].dtype) for key, d in zip(keys, grads)})
    return got


def work(case):
    size = {"f32": 4, "bf16": 2}
    if case["kind"] in ("act", "sequence"):
        h, dk, dv, es = case["heads"], case["dk"], case["dv"], size[case["dtype"]]
        if case["kind"] == "act":
            return {"bytes": case["envs"] * h * (8 * dk * dv + es * (2 * dk + 2 * dv)), "flops": case["envs"] * h * 5 * dk * dv}
        rows, states = case["steps"] * case["envs"] * h, 8 * case["envs"] * h * dk * dv
        if not case["train"]:
            return {"bytes": rows * es * (2 * dk + 2 * dv) + states, "flops": rows * 4 * dk * dv}
        return {"bytes": rows * es * (4 * dk + 4 * dv) + 2 * states, "flops": rows * 14 * dk * dv}
    if case["kind"] == "clip":
        sizes = _sizes(case)
        of = [4, 2] if case["dtype"] == "mixed" else [size[case["dtype"]]]
        held = sum(m * of[(i // 2) % len(of)] for i, m in enumerate(sizes))
        return {"bytes": 2 * held, "flops": 3 * sum(sizes)}
    n, xs, es = case["rows"] * case["width"], size[case["stream"]], size[case["dtype"]]
    if not case["train"]:
        return {"bytes": n * (2 * xs + 3 * es), "flops": 16 * n}
    return {"bytes": n * (4 * xs + 6 * es) + 24 * case["width"], "flops": 50 * n}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"act": _exact_act, "sequence": _exact_sequence, "clip": _exact_clip, "block": _exact_block}[case["kind"]](s)


def _exact_act(s):
    out, state = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda"), s["state"].double()
    lam = s["log_decay"].double().exp().view(1, -1, 1, 1)
    on = ~s["skip"]
    old = state[on]
    old[s["reset"][on]] = 0.0
    new = lam * old + torch.einsum("nhi,nhj->nhij", s["k"][on].double(), s["v"][on].double())
    state[on] = new
    out[on] = s["scale"] * torch.matmul(s["q"][on].double().unsqueeze(-2), new).squeeze(-2)
    return {"out": out, "state": state}


def _exact_sequence(s):
    """The recurrence itself, token by token; its gradients by the recurrence backwards."""
    t, n = s["q"].shape[:2]
    if t * n * s["heads"] * s["dk"] * s["dv"] > 2e10:
        return None
    q, k, v = (s[key].detach().double() for key in ("q", "k", "v"))
    lam, state = s["log_decay"].double().exp().view(1, -1, 1, 1), s["state"].detach().double()
    length = s["lengths"] if s["lengths"] is not None else torch.full((n,), t, device="cuda")
    live = torch.arange(t, device="cuda").unsqueeze(1) < length  # [t, n]
    passes = (~s["reset"]).double()
    out, dq = torch.zeros_like(v), torch.zeros_like(q)
    do = s["dout"].double() if s["train"] else None
    for i in range(t):
        on = live[i].view(n, 1, 1, 1)
        new = lam * passes[i].view(n, 1, 1, 1) * state + k[i].unsqueeze(-1) * v[i].unsqueeze(-2)
        state = torch.where(on, new, state)
        row = torch.matmul(q[i].unsqueeze(-2), state).squeeze(-2)
        out[i] = torch.where(on.squeeze(-1), s["scale"] * row, torch.zeros_like(row))
        if s["train"]:
            row = torch.matmul(state, do[i].unsqueeze(-1)).squeeze(-1)
            dq[i] = torch.where(on.squeeze(-1), s["scale"] * row, torch.zeros_like(row))
    if not s["train"]:
        return {"out": out, "state": state}
    dk, dv, r = torch.zeros_like(k), torch.zeros_like(v), s["dstate"].double()
    for i in reversed(range(t)):
        on = live[i].view(n, 1, 1, 1)
        here = r + s["scale"] * q[i].unsqueeze(-1) * do[i].unsqueeze(-2)
        a, b = torch.matmul(here, v[i].unsqueeze(-1)).squeeze(-1), torch.matmul(k[i].unsqueeze(-2), here).squeeze(-2)
        dk[i], dv[i] = torch.where(on.squeeze(-1), a, torch.zeros_like(a)), torch.where(on.squeeze(-1), b, torch.zeros_like(b))
        r = torch.where(on, lam * passes[i].view(n, 1, 1, 1) * here, r)
    return {"out": out, "state": state, "dq": dq, "dk": dk, "dv": dv, "dstate": r}


def _exact_clip(s):
    flat = [g.double() for g in s["grads"]]
    norm = math.sqrt(math.fsum(float(torch.dot(g, g)) for g in flat))
    by = min(1.0, s["max_norm"] / (norm + EPS))
    return [torch.tensor(norm, dtype=torch.float64)] + [g * by for g in flat]


def _exact_block(s):
    x, b, u, post, res, pre = (s[key].detach().double() for key in ("x", "block", "gate", "post", "res", "pre"))
    width = x.shape[1]
    rb = (b.pow(2).sum(1, keepdim=True) / width + EPS).pow(-0.5)
    sig = torch.sigmoid(u)
    bn = b * rb
    y = x + res * sig * bn * post
    ry = (y.pow(2).sum(1, keepdim=True) / width + EPS).pow(-0.5)
    yn = y * ry
    if not s["train"]:
        return {"y": y, "z": yn * pre}
    dy, dz = s["dy"].double(), s["dz"].double()
    g = dz * pre
    full = dy + ry * (g - yn * (g * yn).sum(1, keepdim=True) / width)
    gb = full * res * sig * post
    db = rb * (gb - bn * (gb * bn).sum(1, keepdim=True) / width)
    du = full * res * bn * post * sig * (1 - sig)
    col = (full * sig * bn).sum(0)
    return {"y": y, "z": yn * pre, "dx": full, "dblock": db, "dgate": du, "dpost": col * res, "dres": col * post, "dpre": (dz * yn).sum(0)}
