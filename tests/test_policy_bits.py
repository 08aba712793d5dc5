"""CPU-only: what the tolerances of tests/policy_bits.py let pass and what not."""
import pytest
import torch

import policy_reference as ref
from policy_bits import attention_bits


def problem(T, N, H, dk, dv, log_decay):
    gen = torch.Generator().manual_seed(T + dk)
    rand = lambda *s: torch.randn(*s, generator=gen).bfloat16()  # noqa: E731
    p = dict(q=rand(T, N, H, dk), k=rand(T, N, H, dk), v=rand(T, N, H, dv), log_decay=torch.full((H,), log_decay), state=rand(N, H, dk, dv).float(), scale=dk**-0.5)
    return p, rand(T, N, H, dv), rand(N, H, dk, dv).float()


@pytest.mark.parametrize("size, log_decay", [((150, 2, 1, 64, 64), -0.06), ((400, 1, 1, 32, 32), -1e-4), ((257, 1, 1, 128, 64), -0.002)], ids=str)
def test_what_passes_and_what_does_not(size, log_decay):
    p, dout, dlast = problem(*size, log_decay)
    want, tol = attention_bits(**p, dout=dout, dlast=dlast)
    for key, w in want.items():
        ref.close(w.bfloat16(), w, tol[key], key)  # rounded once
        for wrong in (0.95 * w, 1.05 * w, (w + 2.0**-8 * w.square().mean().sqrt() * torch.randn(w.shape, generator=torch.Generator().manual_seed(2), dtype=w.dtype))):
            with pytest.raises(AssertionError):
                ref.close(wrong.bfloat16(), w, tol[key], key)
    for tokens in (slice(0, 16), slice(48, 64)):  # a tile of 16 tokens that adds nothing
        part = {**p, "v": p["v"].clone()}
        part["v"][tokens] = 0
        with pytest.raises(AssertionError):
            ref.close(ref.attention(**part)["out"].bfloat16(), want["out"], tol["out"], "out")
    wrong = {**p, "log_decay": p["log_decay"] * 1.1}
    for key, w in ref.attention(**wrong, dout=dout, dlast=dlast).items():
        if key in want:
            with pytest.raises(AssertionError):
                ref.close(w.bfloat16(), want[key], tol[key], key)
