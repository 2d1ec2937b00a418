"""64-bit oracle of rotary positions, from their definition."""

import numpy as np

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step, of the value
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}  # and below the normal range

SHARE = {"f32": 2.0 ** -21, "16": 2.0 ** -19, "8": 2.0 ** -18}


def kind(dtype):
    return "f32" if dtype == "f32" else "16"


def angles(frequencies, positions):
    """(cos, sin) [tokens, 1, pairs]: products and remainders with 64 bits of
    fraction, so those of positions up to 2^30 are good to 2^-34."""
    two_pi = np.longdouble("6.283185307179586476925286766559005768")
    turn = np.asarray(positions).astype(np.longdouble)[:, None] * np.asarray(frequencies, np.float64).astype(np.longdouble)
    a = np.remainder(turn, two_pi).astype(np.float64)[:, None, :]
    return np.cos(a), np.sin(a)


def rotate(rot, x, positions, backward=False, to="f32"):
    """(out, bound) of x [tokens, heads, head_dim] in 64 bits.  ``bound``: how far
    a kernel may be off before its last rounding, as a share of gain (|a| + |b|).

    f32 results: the angle is held to 2^-32 turns; its rest, at most pi / 4, has
    been rounded three times (2.5 * 2^-24 of it: 2^-23), its sine and cosine to
    two steps more (2^-23), the gain, its product with them, and the two products
    and their sum once each: 2^-22 + 4 * 2^-24 < 2^-21.

    16-bit results (``to`` "16"): the angle, at most pi, in f32 (three roundings,
    3 * 2^-24 of pi at most: 2^-20.8), sines and cosines off by 2^-21.2 more as
    CUDA documents them, and the same 4 * 2^-24: 2^-19.7 < 2^-19.

    Keys on their way into 8 bits (``to`` "8"): two such turns one after another,
    the first one of the 16-bit kind (2^-20), the second of the f32 kind (2^-22);
    a turn's error is a vector of at most sqrt 2 of that, and the products that
    join them are rounded by 3 * 2^-24: sqrt 2 * (2^-20 + 2^-22) + 7 * 2^-24
    < 2^-18.9 + 2^-21 < 2^-18."""
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
        bound[..., a] = bound[..., b] = abs(rot.gain) * (np.abs(u) + np.abs(v)) * SHARE[to]
    return out, bound


def close(got, want, bound, dtype):
    """Within the bound and the output's own rounding."""
    tol = bound + HALF[dtype] * (np.abs(want) + bound) + TINY[dtype]
    return bool((np.abs(got.astype(np.float64) - want) <= tol).all())
