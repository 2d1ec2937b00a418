"""64-bit oracle of rotary positions, from their definition."""

import numpy as np

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step, of the value
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}  # and below the normal range


def angles(frequencies, positions):
    """(cos, sin) [tokens, 1, pairs]: products and remainders with 64 bits of
    fraction, so those of positions up to 2^30 are good to 2^-34."""
    two_pi = np.longdouble("6.283185307179586476925286766559005768")
    turn = np.asarray(positions).astype(np.longdouble)[:, None] * np.asarray(frequencies, np.float64).astype(np.longdouble)
    a = np.remainder(turn, two_pi).astype(np.float64)[:, None, :]
    return np.cos(a), np.sin(a)


def rotate(rot, x, positions, backward=False):
    """(out, bound) of x [tokens, heads, head_dim] in 64 bits.  ``bound``: how far
    a kernel may be off that holds angles to 2^-32 turns and computes in f32,
    before its last rounding.  The angle's rest, at most pi / 4, has been rounded
    three times (2.5 * 2^-24 of it: 2^-23), its sine and cosine to two steps more
    (2^-23), the gain, its product with them, and the two products and their sum
    once each: 2^-22 + 4 * 2^-24 < 2^-21 of gain (|a| + |b|)."""
    x = np.asarray(x, np.float64)
    c, s = angles(rot.frequencies, positions)
    if backward:
        s = -s
    r, out, bound = rot.dims, x.copy(), np.zeros(x.shape)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if rot.interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, v = x[..., a], x[..., b]
    with np.errstate(invalid="ignore"):
        out[..., a] = rot.gain * (u * c - v * s)
        out[..., b] = rot.gain * (u * s + v * c)
        bound[..., a] = bound[..., b] = abs(rot.gain) * (np.abs(u) + np.abs(v)) * 2.0 ** -21
    return out, bound


def close(got, want, bound, dtype):
    """Within the bound and the output's own rounding."""
    tol = bound + HALF[dtype] * (np.abs(want) + bound) + TINY[dtype]
    return bool((np.abs(got.astype(np.float64) - want) <= tol).all())
