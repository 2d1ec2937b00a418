"""Rotary positions of queries and keys, and their gradients.

The compiled attention kernels and the key/value cache take queries and keys as
they are; ``Rotary`` turns them to their tokens' positions first.  Its kernel is
hand-written CUDA in ``libemmyrt.so`` (``emmy_rotate`` in ``emmyrt.h``).  The
reference has no counterpart.

    rot = Rotary(head_dim=128, base=500000.0)
    rot.rotate(q, positions, out)             # [tokens, heads, head_dim]; out may be q
    rot.backward(grad_out, positions, grad_q)
    batch.append(layer, k, v, rotary=rot, q=q, q_out=q)    # on the way into a cache

The first ``dims`` values of each head (default all) are pairs (a, b), ``dims`` /
2 apart, or neighbours where ``interleaved``.  Pair i of a token at position p
becomes gain * (a cos(p f) - b sin(p f), a sin(p f) + b cos(p f)) with f =
``frequencies[i]``, by default base ** (-2 i / dims); values behind ``dims`` stay
as they are.  ``scaling`` changes the default for contexts longer than the
trained one, by a ``factor`` s (a dict with its "type"):

* "linear": f / s.
* "base": base * s ** (dims / (dims - 2)) for base.
* "bands": by the turns over the trained ``length`` L, L f / (2 pi): f where
  there are more than ``high`` (4), f / s where fewer than ``low`` (1), between
  them the mixture in proportion.
* "ramp": f up to the pair that makes ``fast`` (32) turns over L, f / s from the
  one that makes ``slow`` (1) on, between them the mixture by index; the gain is
  then 0.1 ln(s) + 1 unless one is given.

Frequencies are held as whole multiples of 2^-64 turns, so that the angle of any
position, however far, is exact to that.  The map is linear and its gradient is
its transpose, ``backward``; a caller whose x was broadcast sums that over the
copies.  Values are turned in f32 and rounded once; sines and cosines are good to
2^-22 of themselves for f32 results, and to 2^-20 for those of 16 bits, so that one
which is small beside the other of its pair may be off by more than its last bit.

Arrays are device arrays as everywhere here (f32, bf16 or f16, last dimension
contiguous, any other strides); positions a device array of int32 or int64, one a
token, or a whole number, the first of consecutive ones.  Calls are queued on
``stream`` (default the device's), return at once and allocate nothing.
"""

from __future__ import annotations

import ctypes as C
import math
import struct
from fractions import Fraction

from .kvcache import _dtype_code, _positions, _stream_of
from .runtime import Device, EmmyError, check, load_library

PAIRS = 256                # EMMY_ROTARY_PAIRS
# 2 pi to 50 digits: a frequency's rounding to 2^-64 turns asks for 20
_TWO_PI = 2 * Fraction("3.1415926535897932384626433832795028841971693993751")
_SCALINGS = {"linear": (), "base": (), "bands": ("length", "low", "high"),
             "ramp": ("length", "fast", "slow")}


class _Rotary(C.Structure):
    """``emmy_rotary``."""
    _fields_ = [("turns", C.c_uint64 * PAIRS), ("gain", C.c_float), ("head_dim", C.c_int32),
                ("dims", C.c_int32), ("interleaved", C.c_int32)]


# emmy_rotate_args: x, out, positions; strides of x and out, position_stride, first,
# tokens; heads, dtype, wide, backward, device (packed at once: a ctypes structure
# costs 2 us more a call)
_ARGS = struct.Struct("@3Q7q5i4x")


def _scaled(dims: int, base: float, scaling) -> tuple[list[float], float]:
    """Frequencies and gain of a scaling."""
    scaling = dict(scaling or {})
    kind = scaling.pop("type", None)
    if kind is None and not scaling:
        return [base ** (-2 * i / dims) for i in range(dims // 2)], 1.0
    if kind not in _SCALINGS:
        raise EmmyError(f"scaling: type must be one of {tuple(_SCALINGS)}, got {kind!r}")
    unknown = set(scaling) - {"factor", *_SCALINGS[kind]}
    if unknown:
        raise EmmyError(f"scaling: {kind} takes no {', '.join(sorted(map(str, unknown)))}")
    for name in ("factor", "length")[:2 if _SCALINGS[kind] else 1]:
        if name not in scaling:
            raise EmmyError(f"scaling: {kind} needs a {name}")
    for name, value in scaling.items():
        if isinstance(value, bool) or not isinstance(value, (int, float)) or not 0 < value < math.inf:
            raise EmmyError(f"scaling: {name} must be a positive number, got {value!r}")
    s = scaling["factor"]
    if kind == "base":
        if dims < 4:
            raise EmmyError("scaling: base needs at least two pairs")
        base *= s ** (dims / (dims - 2))
    f = [base ** (-2 * i / dims) for i in range(dims // 2)]
    if kind == "linear":
        return [x / s for x in f], 1.0
    if kind == "base":
        return f, 1.0
    length = scaling["length"]
    if kind == "bands":
        low, high = scaling.get("low", 1.0), scaling.get("high", 4.0)
        if low >= high:
            raise EmmyError("scaling: low must be below high")
        mix = [min(1.0, max(0.0, (length * x / (2 * math.pi) - low) / (high - low))) for x in f]
        return [(1 - m) * x / s + m * x for m, x in zip(mix, f)], 1.0
    fast, slow = scaling.get("fast", 32.0), scaling.get("slow", 1.0)
    if slow >= fast:
        raise EmmyError("scaling: slow must be below fast")
    if base <= 1:
        raise EmmyError("scaling: ramp needs a base above 1")

    def pair(turns: float) -> float:    # that makes so many turns over the length
        return dims * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))
    low, high = max(0, math.floor(pair(fast))), min(dims - 1, math.ceil(pair(slow)))
    ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 1e-3))) for i in range(dims // 2)]
    return [x * (1 - r) + x / s * r for x, r in zip(f, ramp)], 0.1 * math.log(s) + 1


class Rotary:
    """Rotary positions of heads of ``head_dim`` values.  On no device in
    particular, and the same for every layer, batch and thread."""

    def __init__(self, head_dim: int, dims: int | None = None, base: float = 10000.0,
                 interleaved: bool = False, scaling: dict | None = None, frequencies=None,
                 gain: float | None = None):
        if not 2 <= head_dim <= 2 * PAIRS:
            raise EmmyError(f"head_dim must be between 2 and {2 * PAIRS}, got {head_dim}")
        dims = head_dim if dims is None else dims
        if not 2 <= dims <= head_dim or dims % 2:
            raise EmmyError(f"dims must be even, between 2 and head_dim, got {dims}")
        if frequencies is not None:
            if scaling:
                raise EmmyError("frequencies are given or scaled, not both")
            f, own_gain = [float(x) for x in frequencies], 1.0
            if len(f) != dims // 2:
                raise EmmyError(f"frequencies must be {dims // 2} finite numbers")
        else:
            if not 0 < base < math.inf:
                raise EmmyError(f"base must be a positive number, got {base!r}")
            try:
                f, own_gain = _scaled(dims, float(base), scaling)
            except (OverflowError, ValueError, ZeroDivisionError):
                raise EmmyError("base and scaling give no finite frequencies") from None
        if not all(map(math.isfinite, f)):
            raise EmmyError(f"frequencies must be {dims // 2} finite numbers")
        gain = float(own_gain if gain is None else gain)
        if not math.isfinite(gain) or abs(gain) > 3.4e38:
            raise EmmyError(f"gain must be finite, got {gain!r}")
        self.head_dim, self.dims, self.interleaved = head_dim, dims, bool(interleaved)
        self.frequencies, self.gain = tuple(f), gain
        self._d = _Rotary(gain=gain, head_dim=head_dim, dims=dims, interleaved=self.interleaved)
        for i, x in enumerate(f):
            self._d.turns[i] = round(Fraction(x) * 2 ** 64 / _TWO_PI) % 2 ** 64
        self._ref = C.byref(self._d)

    def rotate(self, x, positions, out, stream=None):
        """Turn ``x`` [tokens, heads, head_dim] to ``positions``, into ``out``
        (same type and shape; ``x`` itself, or no element of it); returns ``out``."""
        return self._turn(x, positions, out, 0, stream)

    def backward(self, grad, positions, out, stream=None):
        """The gradient of ``rotate``'s x from ``grad``, that of its result,
        into ``out``; as ``rotate`` otherwise."""
        return self._turn(grad, positions, out, 1, stream)

    def _turn(self, x, positions, out, backward: int, stream):
        shape, xs, os_ = x.shape, x.stride(), out.stride()
        if len(shape) != 3 or shape[2] != self.head_dim:
            raise EmmyError(f"x has shape {tuple(shape)}, expected [tokens, heads, {self.head_dim}]")
        if out.shape != shape:
            raise EmmyError(f"out has shape {tuple(out.shape)}, expected {tuple(shape)}")
        if xs[2] != 1 or os_[2] != 1:
            raise EmmyError("x and out: the last dimension must be contiguous")
        code = _dtype_code(x.dtype)
        if code > 2 or _dtype_code(out.dtype) != code:
            raise EmmyError("x and out must both be f32, bf16 or f16")
        ordinal, (tokens, heads, _) = x.get_device(), shape
        if ordinal < 0 or out.get_device() != ordinal:
            raise EmmyError("x and out must be on one device")
        at, step, wide, first = _positions(positions, tokens, ordinal)
        st = _stream_of(stream, None if stream is not None else Device.get(ordinal))
        rc = load_library().emmy_rotate(
            self._ref, _ARGS.pack(x.data_ptr(), out.data_ptr(), at, xs[0], xs[1], os_[0], os_[1], step, first,
                                  tokens, heads, code, wide, backward, ordinal), st)
        if rc:
            check(rc, "rotate")
        return out
