"""Rotary positions and rotated appends on the GPU against the 64-bit oracle."""

import threading

import ml_dtypes
import numpy as np
import pytest

from tests import kv8_oracle as kv8
from tests import rotary_oracle as ref
from tests.test_gpu_kvcache import NP, Gpu, cache_of, gpu  # noqa: F401 - gpu is a fixture

pytestmark = pytest.mark.gpu


def values(rng, shape, dtype):
    """Normal values of unlike rows."""
    x = rng.standard_normal(shape) * 2.0 ** rng.integers(-6, 7, shape[:-1] + (1,))
    return x.astype(NP[dtype])


def rotary(head_dim, dims, interleaved, **kw):
    from ptxgen import Rotary
    return Rotary(head_dim, dims, interleaved=interleaved, **kw)


SHAPES = [
    # tokens, heads, head_dim, dims
    (1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 64, 64), (7, 3, 80, 32), (5, 2, 96, 20), (9, 1, 30, 14), (4, 9, 128, 2),
    (2, 4, 512, 512), (33, 4, 128, 126), (2, 67, 64, 48), (300, 2, 64, 16), (1, 300, 256, 256), (13, 1, 7, 6),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_rotate(gpu, shape, interleaved, dtype):  # noqa: F811
    T, H, D, r = shape
    rng = np.random.default_rng(T * D + r)
    rot = rotary(D, r, interleaved, base=500000.0, gain=1.25)
    pos = rng.integers(-1000, 1 << 20, T)
    x = values(rng, (T, H, D), dtype)
    xd, od = gpu.put(x, dtype), gpu.put(np.full((T + 2, H, D), 77).astype(NP[dtype]), dtype)
    from ptxgen import DeviceArray
    view = DeviceArray(od.ptr, dtype, (T, H, D))
    for positions in (gpu.put(pos.astype(np.int32), "i32"), gpu.put(pos.astype(np.int64), "i64")):
        for backward in (False, True):
            call = rot.backward if backward else rot.rotate
            assert call(xd, positions, view) is view
            got = gpu.get(od, (T + 2, H, D), NP[dtype])
            want, bound = ref.rotate(rot, x, pos, backward, ref.kind(dtype))
            assert ref.close(got[:T], want, bound, dtype)
            assert (got[T:].astype(np.float32) == 77).all()
            if D > r:
                assert got[:T, :, r:].tobytes() == x[..., r:].tobytes()
    # in place, and from a first position on, gives the same bits as elsewhere
    call(xd, positions, xd)
    assert gpu.get(xd, x.shape, NP[dtype]).tobytes() == got[:T].tobytes()
    rot.rotate(gpu.put(x, dtype), 12345, view)
    want, bound = ref.rotate(rot, x, 12345 + np.arange(T), to=ref.kind(dtype))
    assert ref.close(gpu.get(view, x.shape, NP[dtype]), want, bound, dtype)


LAYOUTS = [
    # element offset, (token, head) strides of x, then of out, for [6, 3, 32]
    (0, (96, 32), 0, (96, 32)), (1, (97, 32), 0, (96, 32)), (2, (98, 34), 4, (108, 36)), (4, (104, 36), 2, (98, 32)),
    (0, (32, 192), 8, (40, 240)), (0, (0, 32), 0, (96, 32)), (0, (96, 0), 0, (96, 32)), (0, (0, 0), 1, (101, 33)),
    (8, (200, 40), 16, (32, 256)),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved,dims", [(False, 32), (True, 32), (False, 16), (True, 12)])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_strides(gpu, layout, interleaved, dims, dtype):  # noqa: F811
    from ptxgen import DeviceArray
    xo, xs, oo, os_ = layout
    rng = np.random.default_rng(5)
    rot, size = rotary(32, dims, interleaved), 4 if dtype == "f32" else 2
    flat = values(rng, (50, 32), dtype).reshape(-1)
    back = np.full(4000, 77).astype(NP[dtype])
    xd, od = gpu.put(flat, dtype), gpu.put(back, dtype)
    pos = np.array([0, 1, 7, 100, 65535, 9])
    out = DeviceArray(od.ptr + oo * size, dtype, (6, 3, 32), (*os_, 1))
    rot.rotate(DeviceArray(xd.ptr + xo * size, dtype, (6, 3, 32), (*xs, 1)), gpu.put(pos, "i64"), out)
    got = gpu.get(od, back.shape, NP[dtype])
    at = lambda o, s: o + np.arange(6)[:, None, None] * s[0] + np.arange(3)[None, :, None] * s[1] + np.arange(32)  # noqa: E731
    want, bound = ref.rotate(rot, flat[at(xo, xs)], pos, to=ref.kind(dtype))
    assert ref.close(got[at(oo, os_)], want, bound, dtype)
    rest = np.ones(4000, bool)
    rest[at(oo, os_)] = False
    assert (got[rest].astype(np.float32) == 77).all()


def test_slices_of_one_array(gpu):  # noqa: F811
    """Queries and keys of one packed array in place, its values left alone."""
    from ptxgen import DeviceArray
    rng = np.random.default_rng(6)
    rot = rotary(64, 64, False)
    x = values(rng, (9, 4 + 2 + 2, 64), "f16")
    d = gpu.put(x, "f16")
    q, k = (DeviceArray(d.ptr + o * 128, "f16", (9, n, 64), (512, 64, 1)) for o, n in ((0, 4), (4, 2)))
    rot.rotate(q, 5, q)
    rot.rotate(k, 5, k)
    got = gpu.get(d, x.shape, np.float16)
    want, bound = ref.rotate(rot, x, 5 + np.arange(9), to="16")
    assert ref.close(got[:, :6], want[:, :6], bound[:, :6], "f16")
    assert got[:, 6:].tobytes() == x[:, 6:].tobytes()
    # and into a slice behind its own
    out = DeviceArray(d.ptr + 6 * 128, "f16", (9, 2, 64), (512, 64, 1))
    before = got
    rot.backward(k, 5, out)
    got = gpu.get(d, x.shape, np.float16)
    want, bound = ref.rotate(rot, before[:, 4:6], 5 + np.arange(9), True, "16")
    assert ref.close(got[:, 6:], want, bound, "f16") and got[:, :6].tobytes() == before[:, :6].tobytes()


def test_far_positions(gpu):  # noqa: F811
    """Angles stay exact where their f32 products would be whole turns off."""
    rot = rotary(64, 64, False)
    pos = np.array([2 ** 30, 2 ** 30 - 1, -2 ** 30, 987654321, 131071, 0])
    x = np.random.default_rng(8).standard_normal((6, 2, 64)).astype(np.float32)
    out = gpu.put(x, "f32")
    rot.rotate(gpu.put(x, "f32"), gpu.put(pos, "i64"), out)
    want, bound = ref.rotate(rot, x, pos)
    assert ref.close(gpu.get(out, x.shape, np.float32), want, bound, "f32")
    # a period of whole turns: pi / 2 a position, and 2^40 of them
    rot = rotary(2, 2, False, frequencies=[np.pi / 2])
    one = np.array([[[1.0, 0.0]]], np.float32)
    for p, want in ((1, (0, 1)), (2, (-1, 0)), (3, (0, -1)), (4, (1, 0)), (2 ** 30 + 1, (0, 1))):
        out = gpu.put(one, "f32")
        rot.rotate(out, p, out)
        # np.pi is off by 1.2e-16, times the position; the angle by 2^-32 turns
        assert np.abs(gpu.get(out, one.shape, np.float32)[0, 0] - want).max() <= p * 1.3e-16 + 2.0 ** -22


def test_values_that_are_not_finite(gpu):  # noqa: F811
    """They stay in their pairs, and behind dims they are copied."""
    x = np.random.default_rng(9).standard_normal((4, 2, 16)).astype(np.float32)
    x[0, 0, 1], x[1, 1, 3], x[2, 0, 15] = np.inf, np.nan, np.nan
    x[3, 1] = 0.0
    for interleaved in (False, True):
        rot = rotary(16, 12, interleaved)
        out = gpu.put(x, "f32")
        rot.rotate(gpu.put(x, "f32"), 3, out)
        got = gpu.get(out, x.shape, np.float32)
        want, bound = ref.rotate(rot, x, 3 + np.arange(4))
        fine = np.isfinite(want)
        assert ref.close(np.where(fine, got, 0), np.where(fine, want, 0), np.where(fine, bound, 0), "f32")
        assert (np.isfinite(got) == fine).all() and (np.isnan(got) == np.isnan(want)).all()
        assert (got[np.isinf(want)] == want[np.isinf(want)]).all() and (got[3, 1] == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(gpu, interleaved):  # noqa: F811
    """<g, R(x + h d) - R(x - h d)> = 2 h <backward(g), d>: the map is linear, so
    only roundings are between the two (2^-21 of the terms, see the oracle, and
    2^-23 of x h d's)."""
    rng = np.random.default_rng(10)
    rot = rotary(64, 40, interleaved, scaling={"type": "ramp", "factor": 4.0, "length": 512})
    x, d, g = (rng.standard_normal((11, 3, 64)).astype(np.float32) for _ in range(3))
    pos, h = gpu.put(rng.integers(0, 5000, 11), "i64"), np.float32(0.5)
    ends = []
    for y in (x + h * d, x - h * d):
        out = gpu.put(y, "f32")
        ends.append(gpu.get(rot.rotate(out, pos, out), x.shape, np.float32).astype(np.float64))
    out = gpu.put(g, "f32")
    grad = gpu.get(rot.backward(out, pos, out), x.shape, np.float32).astype(np.float64)
    left, right = (g * (ends[0] - ends[1])).sum(), 2 * float(h) * (grad * d).sum()
    size = (np.abs(g) * (np.abs(ends[0]) + np.abs(ends[1]))).sum() + 2 * float(h) * (np.abs(grad) * np.abs(d)).sum()
    assert abs(left - right) <= size * 2.0 ** -20
    # and the gradient is the formula's
    want, bound = ref.rotate(rot, g, gpu.get(pos, 11, np.int64), True)
    assert ref.close(grad, want, bound, "f32")


def test_graph_streams_and_threads(gpu):  # noqa: F811
    """Replays read the positions of the replay; other streams; two threads."""
    import torch
    rot = rotary(128, 128, False)
    x = torch.randn((17, 4, 128), device="cuda", dtype=torch.bfloat16)
    pos, out = torch.arange(17, device="cuda"), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    host = x.float().cpu().numpy().astype(NP["bf16"])

    def check(at):
        want, bound = ref.rotate(rot, host, at, to="16")
        assert ref.close(out.float().cpu().numpy().astype(NP["bf16"]), want, bound, "bf16")
    rot.rotate(x, pos, out, stream=side)
    side.synchronize()
    check(np.arange(17))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rot.rotate(x, pos, out, stream=side)
        rot.backward(out, pos, out, stream=side)
        rot.rotate(x, pos, out, stream=side)
    for shift in (5, 70000):
        pos.copy_(torch.arange(17, device="cuda") + shift)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(np.arange(17) + shift)
    outs = [torch.empty_like(x) for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        for n in range(50):
            rot.rotate(x, 1000 * i + n, outs[i], stream=streams[i])
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(4):
        out = outs[i]
        check(1000 * i + 49 + np.arange(17))


# ---------------------------------------------------------------------------
# appends
# ---------------------------------------------------------------------------


def append_gpu(gpu, case, rot, rng, positions=None, garbage=None):  # noqa: F811
    """One rotated append against the oracle: codes within one rounding of the
    turned values, exponents those of their maxima, queries within theirs."""
    H, G, D, P, dtype, out_dtype, seqs = case
    kv, ql = [a for a, _ in seqs], [b for _, b in seqs]
    T = sum(ql)
    codes, exps = kv8.pool(rng, sum(-(-n // P) for n in kv) + 2, H, P, D)
    table = kv8.tables(rng, len(codes), kv, P)
    k, v = values(rng, (T, H, D), dtype), values(rng, (T, H, D), dtype)
    q = values(rng, (T + 1, H * G, D), dtype)
    if garbage is not None:
        garbage(k, q)
    cache, c, e = cache_of(gpu, codes[None], exps[None])
    batch = cache.batch(table, kv, ql)
    out = gpu.put(np.full(q.shape, 77).astype(NP[out_dtype]), out_dtype)
    place = np.concatenate([np.arange(n - m, n) for n, m in seqs]) if positions is None else positions
    pd = None if positions is None else gpu.put(positions, "i64" if positions.dtype == np.int64 else "i32")
    batch.append(0, gpu.put(k, dtype), gpu.put(v, dtype), rotary=rot, q=gpu.put(q, dtype), q_out=out, positions=pd)
    batch.check_errors()
    got_c, got_e = gpu.get(c, codes.shape, np.uint8), gpu.get(e, exps.shape, np.int8)
    turned, bound = ref.rotate(rot, k.astype(np.float64), place, to="8")
    want_c, want_e = kv8.append(codes, exps, table, kv, ql, turned, v.astype(np.float64))
    assert (got_e == want_e).all()
    assert (got_c[:, 1] == want_c[:, 1]).all()          # values are not turned
    # keys: one rounding, 2^-4 of the value or half of e4m3's least step
    at = 0
    for b, (n, m) in enumerate(seqs):
        for i in range(m):
            page, slot = table[b][(n - m + i) // P], (n - m + i) % P
            for h in range(H):
                unit = 2.0 ** int(got_e[page, 0, h])
                held, y = kv8.DECODE[got_c[page, 0, h, slot]] * unit, turned[at + i, h]
                nan = np.isnan(y)
                assert (np.isnan(held) == nan).all()
                y, held, off = y[~nan], held[~nan], bound[at + i, h][~nan]
                big = np.abs(y) > 448 * unit             # saturated
                assert (np.abs(held[big]) == 448 * unit).all()
                tol = 2.0 ** -4 * (np.abs(y) + off) + unit * 2.0 ** -10 + off
                assert (np.abs(held - y)[~big] <= tol[~big]).all()
        at += m
    old = np.zeros(got_c.shape[:4], bool)                # and no other code changed but the oracle's
    for b, (n, m) in enumerate(seqs):
        for i in range(n - m, n):
            old[table[b][i // P], 0, :, i % P] = True
    assert (got_c[~old] == want_c[~old]).all()
    got_q = gpu.get(out, q.shape, NP[out_dtype])
    want, bound = ref.rotate(rot, q[:T].astype(np.float64), place, to=ref.kind(out_dtype))
    fine = np.isfinite(want)
    assert ref.close(np.where(fine, got_q[:T], 0), np.where(fine, want, 0), np.where(fine, bound, 0), out_dtype)
    assert (np.isnan(got_q[:T]) == np.isnan(want)).all()
    assert (got_q[T:].astype(np.float32) == 77).all()
    batch.close()
    return got_c


APPENDS = [
    # kv heads, group, head_dim, page, dtype, q_out, [(keys, new tokens)]
    (2, 4, 128, 64, "bf16", "bf16", [(1, 1), (64, 1), (65, 1), (700, 1)]),
    (3, 1, 64, 128, "f16", "f16", [(1, 1), (129, 1), (0, 0), (5, 0)]),
    (1, 5, 128, 64, "f32", "bf16", [(33, 1)]),
    (2, 2, 64, 64, "f32", "f32", [(200, 1), (64, 1)]),
    (2, 2, 128, 64, "bf16", "f16", [(130, 70), (64, 64), (3, 2), (65, 0)]),
    (1, 3, 64, 64, "f16", "f16", [(300, 129), (1, 1), (64, 1)]),
    (2, 1, 128, 128, "f32", "f16", [(260, 140), (128, 128)]),
    (1, 2, 64, 256, "bf16", "f32", [(513, 400), (256, 256)]),
    (1, 1, 128, 256, "f32", "bf16", [(300, 299), (20, 7)]),
    (8, 4, 128, 64, "bf16", "bf16", [(900, 900)] * 2 + [(700, 1)]),
]


@pytest.mark.parametrize("dims,interleaved", [(64, False), (64, True), (128, False), (20, False), (34, True), (2, False)])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"h{c[0]}x{c[1]}d{c[2]}p{c[3]}{c[4]}-{c[5]}n{len(c[6])}")
def test_append(gpu, case, dims, interleaved):  # noqa: F811
    rot = rotary(case[2], min(dims, case[2]), interleaved, base=500000.0, gain=0.75)
    append_gpu(gpu, case, rot, np.random.default_rng(11))


@pytest.mark.parametrize("kind", [np.int32, np.int64])
@pytest.mark.parametrize("case", [APPENDS[0], APPENDS[4]], ids=["one", "pages"])
def test_append_positions(gpu, case, kind):  # noqa: F811
    rng = np.random.default_rng(12)
    pos = rng.integers(-50, 1 << 30, sum(m for _, m in case[6])).astype(kind)
    append_gpu(gpu, case, rotary(case[2], 64, False), rng, pos)


@pytest.mark.parametrize("case", [APPENDS[0], APPENDS[4]], ids=["one", "pages"])
def test_append_not_finite(gpu, case):  # noqa: F811
    """NaN and what its pair makes of infinities stay out of the page's scale."""
    def garbage(k, q):
        k[0, 0, 3], k[1, -1, 70], k[2, 0, :] = np.nan, np.inf, np.nan
        q[0, 1, 2], q[3, 0, 5] = np.nan, np.inf
    append_gpu(gpu, case, rotary(case[2], case[2], False), np.random.default_rng(13), garbage=garbage)


def test_append_in_place_of_one_array(gpu):  # noqa: F811
    """q, k and v slices of one array, q turned in place; without q the same codes."""
    from ptxgen import DeviceArray
    rng = np.random.default_rng(14)
    rot = rotary(64, 64, False)
    x = values(rng, (70, 4 + 2 + 2, 64), "bf16")
    codes, exps = kv8.pool(rng, 3, 2, 64, 64)
    results = []
    for with_q in (True, False):
        cache, c, _ = cache_of(gpu, codes[None], exps[None])
        batch = cache.batch([[2, 0]], [75], [70])
        d = gpu.put(x, "bf16")
        q, k, v = (DeviceArray(d.ptr + o * 128, "bf16", (70, n, 64), (512, 64, 1)) for o, n in ((0, 4), (4, 2), (6, 2)))
        batch.append(0, k, v, rotary=rot, **({"q": q, "q_out": q} if with_q else {}))
        batch.check_errors()
        got = gpu.get(d, x.shape, NP["bf16"])
        assert got[:, 4:].tobytes() == x[:, 4:].tobytes()
        if with_q:
            want, bound = ref.rotate(rot, x[:, :4], 5 + np.arange(70), to="16")
            assert ref.close(got[:, :4], want, bound, "bf16")
        results.append(gpu.get(c, codes.shape, np.uint8).tobytes())
        from ptxgen.runtime import EmmyError
        for bad in (k, DeviceArray(d.ptr + 128, "bf16", (70, 4, 64), (512, 64, 1)),
                    DeviceArray(d.ptr, "f16", (70, 4, 64), (512, 64, 1))):
            if bad is k:
                with pytest.raises(EmmyError, match="q_out overlaps"):
                    batch.append(0, k, v, rotary=rot, q=DeviceArray(d.ptr, "bf16", (70, 2, 64), (512, 64, 1)), q_out=k)
            elif bad.ptr != d.ptr:
                with pytest.raises(EmmyError, match="q_out overlaps"):
                    batch.append(0, k, v, rotary=rot, q=q, q_out=bad)
        batch.close()
    assert results[0] == results[1]


def test_append_bad_page(gpu):  # noqa: F811
    """A page outside the pool: reported, its keys left out, queries turned."""
    rng = np.random.default_rng(15)
    from ptxgen.runtime import EmmyError
    rot = rotary(64, 64, False)
    codes, exps = kv8.pool(rng, 3, 1, 64, 64)
    for m in (1, 3):
        cache, c, _ = cache_of(gpu, codes[None], exps[None])
        batch = cache.batch([[0], [1]], [5, 5], [m, m])
        # the table as a graph's owner might have overwritten it
        gpu.dev.htod(batch._d.page_table, np.array([[0], [7]], np.int32))
        k = values(rng, (2 * m, 1, 64), "bf16")
        q = values(rng, (2 * m, 2, 64), "bf16")
        out = gpu.put(np.zeros_like(q), "bf16")
        batch.append(0, gpu.put(k, "bf16"), gpu.put(k, "bf16"), rotary=rot, q=gpu.put(q, "bf16"), q_out=out)
        with pytest.raises(EmmyError, match="outside the pool"):
            batch.check_errors()
        want, bound = ref.rotate(rot, q, np.tile(np.arange(5 - m, 5), 2), to="16")
        assert ref.close(gpu.get(out, q.shape, NP["bf16"]), want, bound, "bf16")
        assert (gpu.get(c, codes.shape, np.uint8)[1:] == codes[1:]).all()
        batch.close()


def test_steps_of_generation(gpu):  # noqa: F811
    """A prompt, then tokens one at a time, rotated on the way into the cache and
    attended over: scores depend on distances alone, so the whole shifted by a
    thousand positions gives the same answers, within twice the codes' rounding
    of one key (2^-4) and the bound of attention."""
    import torch
    from ptxgen import KVCache, KVSequences
    rng = torch.Generator(device="cuda").manual_seed(3)
    H, G, D, n = 2, 4, 64, 130
    x = torch.randn((n + 6, H * G + 2 * H, D), generator=rng, device="cuda").bfloat16()
    rot = rotary(D, D, False, scaling={"type": "bands", "factor": 4.0, "length": 64})
    st = torch.cuda.current_stream().cuda_stream
    outs = []
    for shift in (0, 1000):
        cache = KVCache(pages=6, kv_heads=H, head_dim=D)
        cache.dev.sync()
        seqs = KVSequences(cache)
        a = seqs.new()
        got = []
        for lo, hi in [(0, n)] + [(n + i, n + i + 1) for i in range(6)]:
            batch = seqs.batch([a], [hi - lo], stream=st)
            part = x[lo:hi]
            q, out = torch.empty_like(part[:, :H * G].contiguous()), torch.empty((hi - lo, H * G, D), device="cuda", dtype=torch.bfloat16)
            pos = torch.arange(lo, hi, device="cuda") + shift if shift else None
            batch.append(0, part[:, H * G:H * G + H], part[:, H * G + H:], stream=st, rotary=rot,
                         q=part[:, :H * G], q_out=q, positions=pos)
            batch.attend(0, q, out, stream=st)
            batch.check_errors(stream=st)
            got.append(out)
        outs.append(torch.cat(got).float().cpu().numpy())
        cache.close()
    host = x.double().cpu().numpy()
    q, _ = ref.rotate(rot, host[:, :H * G], np.arange(n + 6))
    k, _ = ref.rotate(rot, host[:, H * G:H * G + H], np.arange(n + 6))
    v = host[:, H * G + H:]
    for h in range(H * G):
        s = q[:, h] @ k[:, h // G].T * D ** -0.5
        # keys rounded by 2^-4 of each value (or half of e4m3's least step, 2^-18 of the
        # page's largest) and queries by 2^-8 move a row's scores by at most `move`, its
        # weights by a factor of e^(2 move); values are rounded as keys, the output to bf16
        size, seen = np.abs(q[:, h]) @ np.abs(k[:, h // G]).T, np.tri(n + 6, dtype=bool)
        small = np.abs(q[:, h]).sum(1, keepdims=True) * np.abs(k).max() * 2.0 ** -18
        move = np.where(seen, (2.0 ** -4 + 2.0 ** -8 + 2.0 ** -12) * size + small, 0).max(1, keepdims=True) * D ** -0.5
        s[~seen] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want, weight = p @ v[:, h // G], p @ np.abs(v[:, h // G])
        held = 2.0 ** -4 * weight + np.abs(v).max() * 2.0 ** -18
        tol = np.expm1(2 * move) * (weight + held) + held
        tol += 2.0 ** -8 * (np.abs(want) + tol) + 2.0 ** -10 * np.abs(v).max()   # weights in f16, bf16 outputs
        for got in outs:
            assert (np.abs(got[:, h] - want) <= tol).all()


def test_append_graph(gpu):  # noqa: F811
    """A captured append replays with the lengths, positions and rows of the replay,
    for single tokens and for pages; rows behind the last sequence stay."""
    import torch
    rng = np.random.default_rng(16)
    H, G, D, P = 2, 2, 64, 64
    rot = rotary(D, 48, False)
    side = torch.cuda.Stream()
    for first, later in (([(70, 1), (3, 1)], [(71, 1), (64, 0)]), ([(70, 60), (3, 3)], [(100, 30), (90, 31)])):
        codes, exps = kv8.pool(rng, 6, H, P, D)
        cache, c, e = cache_of(gpu, codes[None], exps[None])
        gpu.dev.sync()
        table = np.array([[5, 0], [2, 4]], np.int32)
        T = sum(m for _, m in first)
        batch = cache.batch(table, [n for n, _ in first], [m for _, m in first], stream=side)
        k, v = (torch.randn((T, H, D), device="cuda").half() for _ in range(2))
        q, pos = torch.randn((T, H * G, D), device="cuda").half(), torch.zeros(T, dtype=torch.int32, device="cuda")
        out = torch.zeros_like(q)
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            batch.append(0, k, v, stream=side, rotary=rot, q=q, q_out=out, positions=pos)
        assert gpu.get(c, codes.shape, np.uint8).tobytes() == codes.tobytes()
        for seqs, shift in ((first, 0), (later, 1 << 20)):
            gpu.dev.htod(c.ptr, codes)
            gpu.dev.htod(e.ptr, exps)
            gpu.dev.sync()
            n = sum(m for _, m in seqs)
            place = np.concatenate([np.arange(a - b, a) for a, b in seqs]) + shift
            batch.update(table, [a for a, _ in seqs], [b for _, b in seqs], stream=side)
            pos[:n] = torch.from_numpy(place.astype(np.int32)).cuda()
            k.copy_(torch.randn_like(k))
            out.fill_(77)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            batch.check_errors(stream=side)
            want, bound = ref.rotate(rot, q[:n].cpu().numpy(), place, to="16")
            assert ref.close(out[:n].cpu().numpy(), want, bound, "f16") and (out[n:] == 77).all()
            turned, bound = ref.rotate(rot, k[:n].cpu().numpy(), place, to="8")
            want_c, want_e = kv8.append(codes, exps, table, [a for a, _ in seqs], [b for _, b in seqs], turned,
                                        v[:n].cpu().numpy().astype(np.float64))
            got_c, got_e = gpu.get(c, codes.shape, np.uint8), gpu.get(e, exps.shape, np.int8)
            assert (got_e == want_e).all() and (got_c[:, 1] == want_c[:, 1]).all()
            # a code may round to either side of a border that the bound reaches over
            off = np.abs(kv8.DECODE[got_c[:, 0]] - kv8.DECODE[want_c[:, 0]])
            assert (off <= 2.0 ** -3 * np.abs(kv8.DECODE[want_c[:, 0]]) + 2.0 ** -9).all() and (off > 0).mean() < 1e-3
        torch.cuda.synchronize()
        del graph
        batch.close()


def test_many_heads_and_wide_strides(gpu):  # noqa: F811
    """Offsets of rows and heads past 2^31 bytes."""
    import torch
    rot = rotary(8, 8, False)
    x = torch.empty((3, (1 << 30) + 64), dtype=torch.bfloat16, device="cuda")
    step = 1 << 29
    view = x.as_strided((3, 3, 8), ((1 << 30) + 64, step, 1))
    view.copy_(torch.randn((3, 3, 8), device="cuda").bfloat16())
    host = view.float().cpu().numpy()
    out = torch.empty((3, 3, 8), dtype=torch.bfloat16, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    rot.rotate(view, 7, out, stream=st)
    want, bound = ref.rotate(rot, host, 7 + np.arange(3), to="16")
    assert ref.close(out.float().cpu().numpy(), want, bound, "bf16")
    rot.rotate(view, 7, view, stream=st)
    assert (view == out).all()


SLOW = [1e6 ** (-126 / 128) / 32, 1e-9, 3e-11]     # the slowest pair of a stretched context, and slower ones


def slow_bound(angle, positions):
    """f32, small angles: the rest of a turn, 2 pi 2^-64 and their product are rounded
    by 2.5 * 2^-24 of it, the sine's last sum by 2^-24; one times it and nothing times
    the cosine are exact.  The frequency is held to 2^-65 turns."""
    return 2.0 ** -22 * np.abs(angle) + np.abs(positions)[:, None] * 2 * np.pi * 2.0 ** -65


@pytest.mark.parametrize("head_dim,dims,interleaved", [(8, 6, True), (12, 6, True), (7, 6, True), (8, 6, False), (7, 6, False), (12, 8, False)])
def test_slow_frequencies(gpu, head_dim, dims, interleaved):  # noqa: F811
    """Small angles keep f32's precision, and a turn back undoes a turn."""
    fs = (SLOW + [1e-8])[:dims // 2]
    rot = rotary(head_dim, dims, interleaved, frequencies=fs)
    pos = np.array([1, -1, 3, -7, 1000, -999])
    low, high = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, dims // 2), slice(dims // 2, dims))
    x = np.zeros((6, 2, head_dim), np.float32)
    x[..., high] = 1
    out = gpu.put(x, "f32")
    rot.rotate(out, gpu.put(pos, "i64"), out)
    got = gpu.get(out, x.shape, np.float32).astype(np.float64)
    angle = pos[:, None] * np.array(fs)
    tol = slow_bound(angle, pos)[:, None]
    assert (np.abs(got[..., low] + np.sin(angle)[:, None]) <= tol).all()
    assert (np.abs(got[..., high] - np.cos(angle)[:, None]) <= 2.0 ** -22).all()
    # -s c + c s, of the same c and s: each product and the sum once more
    for undo, at in ((rot.rotate, -pos), (rot.backward, pos)):
        back = gpu.put(got.astype(np.float32), "f32")
        undo(back, gpu.put(at, "i64"), back)
        assert (np.abs(gpu.get(back, x.shape, np.float32)[..., low]) <= 2.0 ** -22 * np.abs(angle)[:, None]).all()


def test_slow_frequencies_of_appended_queries(gpu):  # noqa: F811
    """So do queries on the way into f32, of single tokens and of pages."""
    rng = np.random.default_rng(17)
    D, r = 64, 6
    rot = rotary(D, r, False, frequencies=SLOW)
    for ql in ([1, 1, 1], [1, 2, 3]):
        T, places = sum(ql), np.concatenate([np.arange(5, 5 + m) for m in ql])
        codes, exps = kv8.pool(rng, 3, 1, 64, D)
        cache, _, _ = cache_of(gpu, codes[None], exps[None])
        batch = cache.batch([[0], [1], [2]], [5 + m for m in ql], ql)
        q = np.zeros((T, 2, D), np.float32)
        q[..., 3:6] = 1
        k, out = gpu.put(values(rng, (T, 1, D), "f32"), "f32"), gpu.put(q, "f32")
        batch.append(0, k, k, rotary=rot, q=gpu.put(q, "f32"), q_out=out)
        batch.check_errors()
        got = gpu.get(out, q.shape, np.float32).astype(np.float64)
        angle = places[:, None] * np.array(SLOW)
        assert (np.abs(got[..., :3] + np.sin(angle)[:, None]) <= slow_bound(angle, places)[:, None]).all()
        batch.close()


def test_append_most_query_heads(gpu):  # noqa: F811
    """One token of 2^20 query heads, the most there may be, and of 2^18."""
    import torch
    from ptxgen import KVCache
    rot = rotary(64, 64, False)
    st = torch.cuda.current_stream().cuda_stream
    cache = KVCache(pages=2, kv_heads=2, head_dim=64)
    cache.dev.sync()
    k = torch.randn((1, 2, 64), device="cuda").bfloat16()
    for heads in (1 << 18, 1 << 20):
        batch = cache.batch([[1]], [4], stream=st)
        q = torch.randn((1, heads, 64), device="cuda").bfloat16()
        out = torch.zeros_like(q)
        batch.append(0, k, k, stream=st, rotary=rot, q=q, q_out=out)
        batch.check_errors(stream=st)
        # some heads against the oracle, all against the row kernel: each is off by
        # 2^-8 of the value and 2^-19 (|a| + |b|)
        want = torch.empty_like(q)
        rot.rotate(q, 3, want, stream=st)
        some = torch.cat([torch.arange(9), torch.randint(heads, (50,)), torch.arange(heads - 9, heads)])
        value, bound = ref.rotate(rot, q[:, some].float().cpu().numpy(), 3 + np.arange(1), to="16")
        for got in (out, want):
            assert ref.close(got[:, some].float().cpu().numpy(), value, bound, "bf16")
        assert ((out.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 2.0 ** -17 * q.float().abs().max()).all()
        batch.close()
    cache.close()


@pytest.mark.parametrize("dims,interleaved,positions", [(128, False, False), (128, True, False), (64, False, False), (20, False, False), (128, False, True)])
@pytest.mark.parametrize("page,longest,dtype,heads", [(64, 40, "bf16", 8), (64, 40, "f32", 3), (256, 140, "f16", 3)])
def test_append_many_pages(gpu, dims, interleaved, positions, page, longest, dtype, heads):  # noqa: F811
    """More pages than fill the GPU, so that a block takes several keys' and values'
    heads of a page, four of them one after another: 242 places for pages."""
    rng = np.random.default_rng(18)
    lens = [int(n) for n in rng.integers(1, 6, 119)]
    seqs = [(longest + 30, longest)] + [(int(rng.integers(n, page + 40)), n) for n in lens]
    rot = rotary(128, dims, interleaved, base=500000.0)
    T = sum(m for _, m in seqs)
    pos = rng.integers(0, 1 << 20, T) if positions else None
    append_gpu(gpu, (heads, 1, 128, page, dtype, dtype, seqs), rot, rng, pos)
