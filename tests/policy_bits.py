"""How many bits decay attention holds in bfloat16: tolerances that a rounding of a score or of the state to bfloat16 does not meet.

What the inputs hold is exact; between them and a result lie sums in float32 and, of each term once, a score or a state's element as two bfloat16,
the number and what its rounding leaves, each rounded: off by at most 2^-8 * 2^-8 = 2^-16 of it.  With A the recurrence on magnitudes and
n = dk + dv + T + 32 (tests/policy_reference.py: attention_tolerance), a result is rounded to its type once and is off by at most

    2^-8 |want| + (1 + 2^-8) (2^-16 + n 2^-24) A

The terms have both signs, so |want| is far below A: a second rounding of terms to bfloat16 would be allowed 2^-8 A."""
import policy_reference as ref


def attention_bits(q, k, v, log_decay, state=None, reset=None, lengths=None, scale=1.0, dout=None, dlast=None):
    """-> (the reference's results, their tolerances) of the results that have q's type"""
    mag = lambda x: None if x is None else x.detach().double().cpu().abs()  # noqa: E731
    want = ref.attention(q, k, v, log_decay, state, reset, lengths, scale, dout, dlast)
    A = ref.attention(mag(q), mag(k), mag(v), log_decay, mag(state), reset, lengths, abs(scale), mag(dout), mag(dlast))
    n = (q.shape[3] + v.shape[3] + q.shape[0] + 32) * 2.0**-24
    half = ref.HALF[q.dtype]
    keys = [key for key in want if "state" not in key]
    return {key: want[key] for key in keys}, {key: half * want[key].abs() + (1 + half) * (2.0**-16 + n) * A[key] + 1e-37 for key in keys}
