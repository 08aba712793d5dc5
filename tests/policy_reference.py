"""Plain 64-bit implementations of the policy operators (rl4mm_amd/policy_ops.py) and the error that their arithmetic may make.

A rounding to a type is off by at most half a step, eps / 2 relative to the value: HALF below.  A sum of n products in float32 is off by at
most about n * 2^-24 times the sum of the products' magnitudes, which `attention` computes too, by running on magnitudes."""
import torch

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def attention(q, k, v, log_decay, state=None, reset=None, lengths=None, scale=1.0, dout=None, dlast=None):
    """The recurrence, token by token, and its gradients backwards -> dict(out, state[, dq, dk, dv, dstate]); inputs of any type, on any device."""
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    T, N, H, dk = q.shape
    dv = v.shape[3]
    lam = log_decay.detach().double().cpu().exp()[None, :, None, None]
    S = torch.zeros(N, H, dk, dv, dtype=torch.float64) if state is None else state.detach().double().cpu().clone()
    cut = torch.zeros(T, N, dtype=torch.bool) if reset is None else reset.cpu().bool()
    length = torch.full((N,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    out, states = torch.zeros(T, N, H, dv, dtype=torch.float64), []
    for t in range(T):
        on = t < length
        old = torch.where(cut[t][:, None, None, None], torch.zeros_like(S), S)
        S = torch.where(on[:, None, None, None], lam * old + k[t][..., :, None] * v[t][..., None, :], S)
        states.append(S)
        out[t] = torch.where(on[:, None, None], scale * torch.einsum("nhi,nhij->nhj", q[t], S), 0.0)
    got = {"out": out, "state": S}
    if dout is None and dlast is None:
        return got
    do = torch.zeros_like(out) if dout is None else dout.detach().double().cpu()
    R = torch.zeros_like(S) if dlast is None else dlast.detach().double().cpu().clone()
    d = {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    for t in reversed(range(T)):
        on = (t < length)[:, None, None]
        here = R + scale * q[t][..., :, None] * do[t][..., None, :]
        d["dq"][t] = torch.where(on, scale * torch.einsum("nhij,nhj->nhi", states[t], do[t]), 0.0)
        d["dk"][t] = torch.where(on, torch.einsum("nhij,nhj->nhi", here, v[t]), 0.0)
        d["dv"][t] = torch.where(on, torch.einsum("nhij,nhi->nhj", here, k[t]), 0.0)
        passed = torch.where(cut[t][:, None, None, None], torch.zeros_like(R), lam * here)
        R = torch.where(on[..., None], passed, R)
    return {**got, **d, "dstate": R}


def attention_tolerance(q, k, v, log_decay, state=None, reset=None, lengths=None, scale=1.0, dout=None, dlast=None):
    """Per element: how far a result may be from `attention`.  With A the same recurrence on magnitudes:

    float32: every term passes through one dot product over a head, a sum over the tokens, and a decay whose exponent is rounded (a relative 2^-24 per
             64 tokens, and that of the exponential): (dk + dv + T + 32) * 2^-24 * A, and the result's own rounding.
    bfloat16: besides, each score and each state element that multiplies a bfloat16 operand may be rounded to bfloat16 once: 2^-8 * A, and the
             result's own rounding, 2^-8 of its value (at most A, with what is off before it: 2^-8 * (1 + 2^-8) * A).
    The state and its gradient are float32 whatever the inputs are."""
    mag = lambda x: None if x is None else x.detach().double().cpu().abs()  # noqa: E731
    A = attention(mag(q), mag(k), mag(v), log_decay, mag(state), reset, lengths, abs(scale), mag(dout), mag(dlast))
    n = (q.shape[3] + v.shape[3] + q.shape[0] + 32) * 2.0**-24
    half = HALF[q.dtype]
    low = 0.0 if q.dtype == torch.float32 else half
    return {key: a * (n if "state" in key else n + low + half * (1 + low + n)) + 1e-37 for key, a in A.items()}


def block(x, b, gate, post, res, pre, eps, dy=None, dz=None):
    """gated_residual_norm and its gradients -> dict(y, z[, dx, dblock, dgate, dpost, dres, dpre])."""
    x, b, post, res, pre = (t.detach().double().cpu() for t in (x, b, post, res, pre))
    sg = torch.ones_like(b) if gate is None else torch.sigmoid(gate.detach().double().cpu())
    rb = (b.square().mean(-1, keepdim=True) + eps).rsqrt()
    bn = b * rb
    y = x + res * sg * post * bn
    ry = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    yn = y * ry
    got = {"y": y, "z": pre * yn}
    if dy is None and dz is None:
        return got
    dy = torch.zeros_like(y) if dy is None else dy.detach().double().cpu()
    dz = torch.zeros_like(y) if dz is None else dz.detach().double().cpu()
    g = dz * pre
    f = dy + ry * (g - yn * (g * yn).mean(-1, keepdim=True))
    e = f * res * sg * post
    got.update(dx=f, dblock=rb * (e - bn * (e * bn).mean(-1, keepdim=True)), dpre=(dz * yn).reshape(-1, x.shape[-1]).sum(0))
    if gate is not None:
        got["dgate"] = f * res * bn * post * sg * (1 - sg)
    m = (f * sg * bn).reshape(-1, x.shape[-1]).sum(0)
    got.update(dpost=res * m, dres=post * m)
    return got


def block_tolerance(x, b, gate, post, res, pre, eps, dy=None, dz=None):
    """Per element.  A row's sums are of `width` terms of one sign (the two mean squares) or of both (the two others, bounded by Cauchy-Schwarz: a mean of
    products with a normed row is at most the root mean square of the other factor); a float32 sum of W terms is off by at most W * 2^-24 of their
    magnitudes, the exponential, division and root by 8 steps in all.  c = (W + 64) * 2^-24 covers every factor of a product once; y and f add two and
    three such terms.  The results' own rounding to their type comes on top."""
    r = block(x, b, gate, post, res, pre, eps, dy, dz)
    X, post, res, pre = (t.detach().double().cpu().abs() for t in (x, post, res, pre))
    B = b.detach().double().cpu()
    W = X.shape[-1]
    c = (W + 64) * 2.0**-24
    sg = torch.ones_like(B) if gate is None else torch.sigmoid(gate.detach().double().cpu())
    rb = (B.square().mean(-1, keepdim=True) + eps).rsqrt()
    bn = B.abs() * rb
    Y = X + res * sg * post * bn  # magnitude of y's terms
    ry = (r["y"].square().mean(-1, keepdim=True) + eps).rsqrt()
    yn = Y * ry
    rms = lambda t: t.square().mean(-1, keepdim=True).sqrt()  # noqa: E731
    worse = 1 + rms(Y) * ry  # how much larger y's terms are than y: errors of y reach the norm with it
    hx, hb = HALF[x.dtype], HALF[b.dtype]
    tol = {"y": 2 * c * Y + hx * r["y"].abs(), "z": 4 * c * worse * pre * yn + hb * r["z"].abs()}
    if dy is None and dz is None:
        return {k: t + 1e-37 for k, t in tol.items()}
    dy = torch.zeros_like(Y) if dy is None else dy.detach().double().cpu().abs()
    dz = torch.zeros_like(Y) if dz is None else dz.detach().double().cpu().abs()
    g = dz * pre
    F = dy + ry * (g + yn * rms(yn) * rms(g))
    E = F * res * sg * post
    ef = 8 * c * worse * F  # error of f
    tol["dx"] = ef + hx * r["dx"].abs()
    tol["dblock"] = rb * (8 * c * worse * 2 * E + bn * 8 * c * worse.amax() * 2 * rms(E) * rms(bn)) + rb * 8 * c * (E + bn * rms(E)) + hb * r["dblock"].abs()
    if gate is not None:
        tol["dgate"] = 10 * c * worse * F * res * bn * post * sg * (1 - sg) + sg * (F * res * bn * post) * 2.0**-22 + hb * r["dgate"].abs()
    rows = F.reshape(-1, W).shape[0]
    flat = lambda t: t.reshape(-1, W).sum(0)  # noqa: E731
    m = flat((10 * c * worse + (rows + 8) * 2.0**-24) * F * sg * bn)
    tol["dpost"], tol["dres"] = res * m, post * m
    tol["dpre"] = flat((6 * c * worse + (rows + 8) * 2.0**-24) * dz * yn)
    return {k: t + 1e-37 for k, t in tol.items()}


def close(got, want, tolerance, what=""):
    """Every element within its tolerance; names the first that is not."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= tolerance)
    if bad.any():
        i = tuple(int(j) for j in bad.nonzero()[0])
        worst = (off / tolerance).nan_to_num(nan=float("inf")).max().item()
        raise AssertionError(f"{what}{list(i)}: {got[i].item()!r} instead of {want[i].item()!r}, {off[i].item():.3g} off where {tolerance[i].item():.3g} is allowed ({int(bad.sum())} of {bad.numel()} elements; worst {worst:.3g} x)")
