"""Rotary positions on the CPU: frequencies of each scaling against their
formulas, how they are held, what the calls refuse, and what they hand on."""

import ctypes as C
import math
from fractions import Fraction
from types import SimpleNamespace

import numpy as np
import pytest

from ptxgen import Rotary, kvcache as kv, rotary as ro
from ptxgen.kvcache import DeviceArray
from ptxgen.runtime import EmmyError
from tests.test_kvcache import dev, small  # noqa: F401 - a fixture


def test_default_frequencies():
    rot = Rotary(128)
    assert rot.dims == 128 and rot.gain == 1.0 and not rot.interleaved
    assert np.allclose(rot.frequencies, 10000.0 ** (-np.arange(64) / 64), rtol=1e-15)


@pytest.mark.parametrize("dims,base", [(2, 10000.0), (64, 500000.0), (30, 1e6), (128, 7.5)])
def test_linear_and_base(dims, base):
    i = np.arange(dims // 2)
    got = Rotary(128, dims, base, scaling={"type": "linear", "factor": 8}).frequencies
    assert np.allclose(got, base ** (-2 * i / dims) / 8, rtol=1e-14)
    if dims > 2:
        got = Rotary(128, dims, base, scaling={"type": "base", "factor": 4.0}).frequencies
        assert np.allclose(got, (base * 4.0 ** (dims / (dims - 2))) ** (-2 * i / dims), rtol=1e-13)
        # the fastest pair as it was, the slowest slowed by the factor
        assert got[0] == 1.0 and math.isclose(got[-1], base ** (-2 * i[-1] / dims) / 4, rel_tol=1e-12)


def test_bands():
    rot = Rotary(128, base=500000.0, scaling={"type": "bands", "factor": 8.0, "length": 8192})
    for i, f in enumerate(rot.frequencies):
        plain = 500000.0 ** (-i / 64)
        wave = 2 * math.pi / plain
        if wave < 8192 / 4:
            want = plain
        elif wave > 8192:
            want = plain / 8
        else:
            mix = (8192 / wave - 1) / 3
            want = (1 - mix) * plain / 8 + mix * plain
        assert math.isclose(f, want, rel_tol=1e-12)
    assert rot.gain == 1.0


def test_ramp():
    s = {"type": "ramp", "factor": 16, "length": 4096}
    rot = Rotary(128, scaling=s)
    assert math.isclose(rot.gain, 0.1 * math.log(16) + 1)
    assert Rotary(128, scaling=s, gain=1.0).gain == 1.0
    plain = 10000.0 ** (-np.arange(64) / 64)
    ratio = np.array(rot.frequencies) / plain
    turns = 4096 * plain / (2 * math.pi)
    assert np.allclose(ratio[turns > 33], 1) and np.allclose(ratio[turns < 0.8], 1 / 16)
    assert (np.diff(ratio) <= 1e-15).all()


def test_turns_hold_frequencies():
    """2^-65 turns at most from f / (2 pi), whatever f is, also whole turns and signs."""
    fs = [1.0, -1.0, 1e-30, 2 * math.pi, 100.0, 3.7e-5]
    rot = Rotary(64, 12, frequencies=fs)
    pi = Fraction("3.1415926535897932384626433832795028841971693993751")
    for t, f in zip(rot._d.turns, fs):
        off = (Fraction(t, 2 ** 64) - Fraction(f) / (2 * pi)) % 1
        assert min(off, 1 - off) <= Fraction(1, 2 ** 65) + Fraction(1, 2 ** 100)
    assert all(t == 0 for t in rot._d.turns[6:])


@pytest.mark.parametrize("kw,says", [
    ({"head_dim": 1}, "head_dim"), ({"head_dim": 514}, "head_dim"), ({"dims": 0}, "dims"),
    ({"dims": 3}, "dims"), ({"dims": 66}, "dims"), ({"base": 0.0}, "base"), ({"base": -5.0}, "base"),
    ({"base": math.inf}, "base"), ({"base": math.nan}, "base"), ({"base": 1e-308, "scaling": {"type": "linear", "factor": 1e-300}}, "finite"),
    ({"scaling": {"type": "what", "factor": 2}}, "type"), ({"scaling": {"factor": 2}}, "type"),
    ({"scaling": {"type": "linear"}}, "needs a factor"),
    ({"scaling": {"type": "bands", "factor": 2}}, "needs a length"),
    ({"scaling": {"type": "linear", "factor": 0}}, "positive"),
    ({"scaling": {"type": "linear", "factor": "2"}}, "positive"),
    ({"scaling": {"type": "linear", "factor": True}}, "positive"),
    ({"scaling": {"type": "linear", "factor": 2, "length": 5}}, "takes no length"),
    ({"scaling": {"type": "bands", "factor": 2, "length": 5, "low": 4.0}}, "below high"),
    ({"scaling": {"type": "ramp", "factor": 2, "length": 5, "slow": 40}}, "below fast"),
    ({"scaling": {"type": "ramp", "factor": 2, "length": 5}, "base": 1.0}, "above 1"),
    ({"scaling": {"type": "base", "factor": 2}, "dims": 2}, "two pairs"),
    ({"frequencies": [1.0]}, "32 finite"), ({"frequencies": [math.nan] * 32}, "finite"),
    ({"frequencies": [1.0] * 32, "scaling": {"type": "linear", "factor": 2}}, "not both"),
    ({"gain": math.nan}, "gain"), ({"gain": 1e39}, "gain"),
])
def test_refusals(kw, says):
    with pytest.raises(EmmyError, match=says):
        Rotary(**{"head_dim": 64, **kw})


@pytest.mark.parametrize("kw", [{"length": 1e-300, "fast": 1e300}, {"length": 5, "fast": 1e308, "slow": 1e307, "factor": 1e-308},
                                {"length": 1e308, "slow": 1e-308}])
def test_ramps_past_all_numbers(kw):
    """Refused as other numbers that give no frequencies, or fine."""
    try:
        rot = Rotary(64, scaling={"type": "ramp", "factor": 2.0, **kw})
    except EmmyError as error:
        assert "finite" in str(error)
    else:
        assert all(map(math.isfinite, rot.frequencies))


@pytest.fixture
def lib(dev, monkeypatch):  # noqa: F811
    monkeypatch.setattr(ro, "load_library", lambda: dev.L)
    return dev.L


def arr(shape, dtype="bf16", ptr=4096, strides=None, device=0):
    return DeviceArray(ptr, dtype, shape, strides, device)


X = (5, 3, 64)


@pytest.mark.parametrize("x,pos,out,says", [
    (arr((5, 3, 80)), 0, arr((5, 3, 80)), "expected"), (arr((5, 64)), 0, arr((5, 64)), "expected"),
    (arr(X), 0, arr((5, 4, 64)), "expected"), (arr(X), 0, arr(X, "f32"), "both"),
    (arr(X, "u8"), 0, arr(X, "u8"), "both"), (arr(X, strides=(384, 128, 2)), 0, arr(X), "contiguous"),
    (arr(X), 0, arr(X, strides=(384, 128, 2)), "contiguous"), (arr(X), 0, arr(X, device=1), "one device"),
    (arr(X), arr((4,), "i32"), arr(X), "positions has shape"), (arr(X), arr((5, 1), "i32"), arr(X), "positions has shape"),
    (arr(X), arr((5,), "f32"), arr(X), "int32 or int64"), (arr(X), arr((5,), "i64", device=1), arr(X), "not on device"),
    (arr(X), np.arange(5), arr(X), "whole number"), (arr(X), None, arr(X), "whole number"),
    (arr(X), 1.5, arr(X), "whole number"), (arr(X), [1, 2, 3, 4, 5], arr(X), "whole number"),
    (arr(X), 2 ** 63 - 3, arr(X), "64 bits"),
])
def test_rotate_refusals(lib, x, pos, out, says):
    for call in (Rotary(64).rotate, Rotary(64).backward):
        with pytest.raises(EmmyError, match=says):
            call(x, pos, out)
    assert not lib.calls


def unpacked(form, raw, names):
    return SimpleNamespace(**dict(zip(names.split(), form.unpack(raw))))


def test_rotate_hands_on(lib):
    rot = Rotary(64, 32, interleaved=True)
    out = arr(X, ptr=8192)
    assert rot.backward(arr(X, strides=(640, 128, 1)), arr((9,), "i32", 512, (2,)), out, stream=11) is out
    (name, (ref, args, st)), = lib.calls
    a = unpacked(ro._ARGS, args, "x out positions x_t x_h out_t out_h position_stride first tokens heads dtype wide backward device")
    assert (name, st, ref._obj.dims, ref._obj.interleaved) == ("emmy_rotate", 11, 32, 1)
    assert (a.x, a.out, a.positions, a.x_t, a.x_h, a.out_t, a.out_h) == (4096, 8192, 512, 640, 128, 192, 64)
    assert (a.position_stride, a.wide, a.tokens, a.heads, a.dtype, a.backward) == (2, 0, 5, 3, 1, 1)
    rot.rotate(out, np.int64(-7), out)
    a = ro._ARGS.unpack(lib.calls[-1][1][1])
    assert (a[2], a[8], a[13], lib.calls[-1][1][2]) == (0, -7, 0, 7)


KV, Q = (5, 2, 64), (5, 6, 64)


@pytest.mark.parametrize("kw,says", [
    ({"rotary": 5}, "rotary is for"), ({"rotary": Rotary(128)}, "of 128 values"),
    ({"q": arr(Q)}, "for a rotary"), ({"positions": arr((5,), "i32")}, "for a rotary"),
    ({"rotary": Rotary(64), "q": arr(Q)}, "together"), ({"rotary": Rotary(64), "q_out": arr(Q)}, "together"),
    ({"rotary": Rotary(64), "q": arr(Q, "f16"), "q_out": arr(Q)}, "keys' type"),
    ({"rotary": Rotary(64), "q": arr(Q), "q_out": arr(Q, "u8")}, "keys' type"),
    ({"rotary": Rotary(64), "q": arr(Q), "q_out": arr((5, 5, 64))}, "q_out has shape"),
    ({"rotary": Rotary(64), "q": arr((4, 6, 64)), "q_out": arr(Q)}, "q has shape"),
    ({"rotary": Rotary(64), "positions": arr((4,), "i32")}, "positions has shape"),
    ({"rotary": Rotary(64), "positions": 7}, "device array"),
    ({"rotary": Rotary(64), "positions": arr((5,), "f32")}, "int32 or int64"),
])
def test_append_refusals(dev, kw, says):  # noqa: F811
    batch = small(dev).batch([[1]], [9], [5])
    with pytest.raises(EmmyError, match=says):
        batch.append(0, arr(KV), arr(KV), **kw)
    assert not any(n.startswith("emmy_kv8_append") for n, _ in dev.L.calls)


def test_append_hands_on(dev):  # noqa: F811
    batch = small(dev).batch([[1]], [9], [5], stream=3)
    rot = Rotary(64, 20)
    batch.append(1, arr(KV), arr(KV, ptr=8192), rotary=rot, q=arr(Q, ptr=512), q_out=arr(Q, "f16", 1024),
                 positions=arr((5,), "i64", 64), stream=3)
    name, a = dev.L.calls[-1]
    assert name == "emmy_kv8_append_rotated" and a[1:4] == (4096, 8192, 1) and a[6] is rot._ref and a[8] == 3
    assert kv._ROTATED.unpack(a[7]) == (64, 512, 1024, 1, 384, 64, 384, 64, 1, 6, 2)
    batch.append(1, arr(KV), arr(KV, ptr=8192), rotary=rot, stream=3)
    assert kv._ROTATED.unpack(dev.L.calls[-1][1][7]) == (0,) * 11


def real():
    from ptxgen.runtime import load_library
    return load_library()


class RotateArgs(C.Structure):
    """``emmy_rotate_args``."""
    _fields_ = [("x", C.c_uint64), ("out", C.c_uint64), ("positions", C.c_uint64),
                ("x_strides", C.c_int64 * 2), ("out_strides", C.c_int64 * 2),
                ("position_stride", C.c_int64), ("first", C.c_int64), ("tokens", C.c_int64),
                ("heads", C.c_int32), ("dtype", C.c_int32), ("wide", C.c_int32),
                ("backward", C.c_int32), ("device", C.c_int32)]


def rotate_args(**kw):
    a = RotateArgs(4096, 1 << 20, 0, (128, 64), (128, 64), 0, 0, 5, 2, 1, 0, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_packed_arguments():
    """The packed form lies as the structure does."""
    values = (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15)
    a = RotateArgs.from_buffer_copy(ro._ARGS.pack(*values))
    assert C.sizeof(RotateArgs) == ro._ARGS.size
    assert (a.x, a.out, a.positions, *a.x_strides, *a.out_strides, a.position_stride, a.first, a.tokens, a.heads,
            a.dtype, a.wide, a.backward, a.device) == values


@pytest.mark.parametrize("kw,says", [
    ({"dtype": 3}, "dtype"), ({"device": -1}, "device"), ({"tokens": -1}, "tokens"), ({"tokens": 2 ** 31}, "tokens"),
    ({"heads": -1}, "heads"), ({"heads": 2 ** 20 + 1}, "heads"), ({"x": 0}, "null"), ({"out": 0}, "null"),
    ({"x": 4097}, "aligned"), ({"out": 4097}, "aligned"), ({"positions": 6}, "positions must"),
    ({"positions": 4, "wide": 1}, "positions must"), ({"x_strides": (C.c_int64 * 2)(-128, 64)}, "negative"),
    ({"out_strides": (C.c_int64 * 2)(127, 64)}, "rows of out"), ({"out_strides": (C.c_int64 * 2)(128, 0)}, "rows of out"),
    ({"out": 4096 + 64}, "x and out overlap"), ({"out": 4096, "x_strides": (C.c_int64 * 2)(256, 64)}, "x and out overlap"),
    ({"x": 1 << 20, "x_strides": (C.c_int64 * 2)(0, 64)}, "x and out overlap"),
])
def test_library_refusals(kw, says):
    """The C entry itself, before it touches a device."""
    L, rot = real(), Rotary(64)
    assert L.emmy_rotate(rot._ref, C.byref(rotate_args(**kw)), None) == -3
    assert says.encode() in L.emmy_last_error()


@pytest.mark.parametrize("field,value,says", [
    ("head_dim", 0, "head_dim"), ("head_dim", 513, "head_dim"), ("dims", 0, "dims"), ("dims", 7, "dims"),
    ("dims", 66, "dims"), ("gain", math.inf, "gain"),
])
def test_library_refuses_rotary(field, value, says):
    L, d = real(), ro._Rotary.from_buffer_copy(Rotary(64)._d)
    setattr(d, field, value)
    assert L.emmy_rotate(C.byref(d), C.byref(rotate_args()), None) == -3
    assert says.encode() in L.emmy_last_error()
    assert L.emmy_rotate(None, C.byref(rotate_args()), None) == -3
    assert L.emmy_rotate(Rotary(64)._ref, None, None) == -3


def test_library_accepts_nothing_to_do():
    L, rot = real(), Rotary(64)
    assert L.emmy_rotate(rot._ref, C.byref(rotate_args(tokens=0, x=0, out=0)), None) == 0
    assert L.emmy_rotate(rot._ref, C.byref(rotate_args(heads=0, x=0, out=0)), None) == 0


class RotatedArgs(C.Structure):
    """``emmy_kv8_rotated_args``."""
    _fields_ = [("positions", C.c_uint64), ("q", C.c_uint64), ("q_out", C.c_uint64), ("position_stride", C.c_int64),
                ("q_strides", C.c_int64 * 2), ("out_strides", C.c_int64 * 2), ("wide", C.c_int32), ("heads", C.c_int32),
                ("out_dtype", C.c_int32)]


def test_packed_append_arguments():
    a = RotatedArgs.from_buffer_copy(kv._ROTATED.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11))
    assert C.sizeof(RotatedArgs) == kv._ROTATED.size
    assert (a.positions, a.q, a.q_out, a.position_stride, *a.q_strides, *a.out_strides, a.wide, a.heads, a.out_dtype) \
        == tuple(range(1, 12))


def two(a, b):
    return (C.c_int64 * 2)(a, b)


@pytest.mark.parametrize("kw,says", [
    ({"positions": 6}, "positions must"), ({"positions": 4, "wide": 1}, "positions must"),
    ({"heads": -1}, "heads"), ({"heads": 2 ** 20 + 1}, "heads"), ({"q": 0}, "null q"), ({"q_out": 0}, "null q"),
    ({"out_dtype": 3}, "q_out must"), ({"q": 4096 + 8}, "16 bytes"), ({"q_out": (1 << 20) + 8}, "16 bytes"),
    ({"q_strides": two(260, 64)}, "16 bytes"), ({"out_strides": two(256, 68)}, "16 bytes"),
    ({"q_strides": two(-256, 64)}, "negative"), ({"out_strides": two(64, 64)}, "rows of q_out"),
    ({"q_out": 4096 + 128}, "q_out overlaps"), ({"q_out": 4096, "out_dtype": 2}, "q_out overlaps"),
    ({"q_out": 4096, "out_strides": two(512, 64)}, "q_out overlaps"),
    ({"q_out": 1 << 24}, "q_out overlaps"), ({"q_out": (1 << 25) - 64}, "q_out overlaps"),      # k, v
])
def test_library_append_refusals(kw, says):
    """The C entry itself, before it touches a device: q and q_out of 4 heads."""
    L = real()
    cache = kv._Cache(codes=4096, exps=4096, page_table=4096, kv_lens=4096, q_starts=4096, status=0, device=0,
                      pages=9, kv_heads=2, head_dim=64, page_size=64, seqs=4, table_width=2, tokens=4, max_q=1)
    a = RotatedArgs(0, 4096, 1 << 20, 0, two(256, 64), two(256, 64), 0, 4, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    rot, st = Rotary(64), two(128, 64)
    call = lambda cache, rot, a: L.emmy_kv8_append_rotated(C.byref(cache), 1 << 24, 1 << 25, 1, st, st, rot, a, None)  # noqa: E731
    assert call(cache, rot._ref, C.byref(a)) == -3 and says.encode() in L.emmy_last_error()
    for bad in (None, Rotary(128)._ref):
        assert call(cache, bad, C.byref(a)) == -3 and b"rotary" in L.emmy_last_error()
    assert call(cache, rot._ref, None) == -3
    cache.tokens = cache.max_q = 0          # nothing to do
    if says in ("16 bytes", "q_out must", "null q", "negative", "rows of q_out", "q_out overlaps"):
        assert call(cache, rot._ref, C.byref(a)) == 0
