"""The paged 8-bit cache on the GPU against the 64-bit oracle: append bit for
bit, attend within the derived bound, page copies bit for bit, and a decoding
run of all of them together."""

import ml_dtypes
import numpy as np
import pytest

from tests import kv8_oracle as ref

pytestmark = pytest.mark.gpu

NP = {"f32": np.float32, "f16": np.float16, "bf16": ml_dtypes.bfloat16}


class Gpu:
    """Host arrays to device arrays and back, on the framework's stream."""

    def __init__(self):
        from ptxgen.runtime import Device
        self.dev = Device.get(0)
        self.ptrs = []

    def put(self, a, dtype, strides=None, shape=None):
        from ptxgen import DeviceArray
        a = np.ascontiguousarray(a)
        p = self.dev.alloc(a.nbytes)
        self.ptrs.append(p)
        self.dev.htod(p, a)
        return DeviceArray(p, dtype, shape or a.shape, strides)

    def get(self, arr, shape, dtype):
        out = np.empty(shape, dtype)
        self.dev.dtoh(out, arr.data_ptr())
        self.dev.sync()
        return out

    def close(self):
        self.dev.sync()
        for p in self.ptrs:
            self.dev.free(p)


@pytest.fixture
def gpu():
    g = Gpu()
    yield g
    g.close()


def cache_of(gpu, codes, exps):
    from ptxgen import KVCache
    lay, n, _, h, p, d = codes.shape
    c, e = gpu.put(codes, "u8"), gpu.put(exps, "i8")
    return KVCache(n, h, d, page_size=p, layers=lay, storage=(c, e)), c, e


def attend_gpu(gpu, codes, exps, table, kv, q_lens, q, dtype, pad=0, **kw):
    """Output rows (and `pad` rows behind them) of one attend call."""
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    batch = cache.batch(table, kv, q_lens)
    rows, heads, d = q.shape
    full = np.concatenate([q, np.ones((pad, heads, d), q.dtype)]) if pad else q
    qd = gpu.put(full, dtype)
    fill = np.full((rows + pad, heads, d), 77.0).astype(NP[dtype])
    od = gpu.put(fill, dtype)
    assert batch.attend(0, qd, od, **kw) is od
    out = gpu.get(od, fill.shape, NP[dtype])
    batch.check_errors()
    again = gpu.put(fill, dtype)
    batch.attend(0, qd, again, **kw)
    assert gpu.get(again, fill.shape, NP[dtype]).tobytes() == out.tobytes()   # no order of arrival in it
    batch.close()
    assert (out[rows:].astype(np.float32) == 77.0).all()
    return out[:rows]


CASES = [
    # kv heads, group, head_dim, page, dtype, window, sinks, [(keys, new tokens)]
    (2, 4, 128, 64, "bf16", 0, 0, [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1), (129, 1)]),
    (1, 8, 64, 64, "f16", 0, 0, [(1, 1), (500, 1), (64, 1)]),
    (3, 1, 128, 128, "f16", 0, 0, [(127, 1), (128, 1), (129, 1), (300, 1)]),
    (1, 16, 128, 256, "bf16", 0, 0, [(700, 1), (255, 1), (257, 1)]),
    (2, 7, 64, 64, "bf16", 0, 0, [(100, 3), (3, 3), (70, 2), (64, 1)]),
    (1, 5, 128, 64, "bf16", 0, 0, [(200, 5), (5, 5), (66, 4)]),
    (1, 32, 64, 64, "bf16", 0, 0, [(130, 1), (1, 1)]),
    (1, 40, 128, 64, "f16", 0, 0, [(90, 1), (190, 2)]),
    (2, 4, 128, 64, "bf16", 16, 0, [(100, 1), (10, 1), (16, 1), (17, 1), (80, 3)]),
    (2, 4, 64, 64, "bf16", 100, 4, [(300, 1), (101, 1), (104, 1), (105, 2), (64, 1), (230, 3)]),
    (1, 2, 128, 64, "f16", 1, 70, [(300, 2), (64, 1), (150, 4)]),
    (1, 2, 64, 64, "f16", 3, 1, [(400, 7), (129, 1)]),
    (1, 8, 128, 64, "bf16", 0, 0, [(9000, 1)]),                      # one sequence in many parts
    (1, 4, 64, 128, "f16", 0, 0, [(5000, 4), (0, 0), (3, 0), (1, 1)]),   # sequences that sit the step out
    # prompts
    (1, 4, 128, 64, "bf16", 0, 0, [(90, 90)]),
    (2, 2, 64, 64, "f16", 0, 0, [(200, 150), (64, 64), (1, 1), (65, 33)]),
    (1, 3, 128, 64, "bf16", 40, 5, [(333, 200), (20, 20)]),
    (1, 1, 64, 128, "bf16", 64, 64, [(400, 300)]),
    (2, 8, 128, 64, "bf16", 0, 0, [(1000, 70), (130, 130), (600, 1)]),
    # few rows and many keys: units cut along the keys
    (1, 4, 128, 64, "bf16", 0, 0, [(3000, 40)]),
    (1, 8, 64, 128, "f16", 1700, 5, [(5000, 30)]),
    (2, 2, 64, 64, "bf16", 0, 0, [(2500, 33), (1200, 150), (900, 1), (700, 2)]),
    # blocks of rows
    (1, 17, 64, 64, "f16", 0, 0, [(300, 1), (40, 1)]),
    (2, 6, 128, 64, "f16", 30, 2, [(700, 5), (90, 3), (64, 1)]),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"h{c[0]}x{c[1]}d{c[2]}p{c[3]}{c[4]}w{c[5]}s{c[6]}n{len(c[7])}")
def test_attend(gpu, case):
    H, G, D, P, dtype, window, sinks, seqs = case
    rng = np.random.default_rng(7)
    kv, ql = [a for a, _ in seqs], [b for _, b in seqs]
    pages = sum(-(-n // P) for n in kv) + 2
    codes, exps = ref.pool(rng, pages, H, P, D)
    table = ref.tables(rng, pages, kv, P)
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP[dtype])
    got = attend_gpu(gpu, codes, exps, table, kv, ql, q, dtype, pad=3, window=window, sinks=sinks)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5, window, sinks)
    assert ref.close(got, want, bound, dtype)


@pytest.mark.parametrize("D,G,window,sinks,seqs", [
    (128, 4, 0, 0, [(n, 1) for n in (1, 2, 31, 33, 64, 65, 400, 1000)]),
    (64, 4, 33, 2, [(n, 1) for n in (1, 33, 34, 35, 36, 64, 97, 98, 400)]),
    (128, 2, 64, 65, [(400, 9), (64, 20), (129, 5)]),
    (64, 8, 5, 0, [(300, 60), (64, 64), (70, 65)]),
    (128, 8, 200, 3, [(1500, 300), (77, 77)]),
    (64, 1, 0, 0, [(700, 513)]),
])
def test_every_key_counts_once(gpu, D, G, window, sinks, seqs):
    """Queries of zero weigh every visible key alike, and key j holds 1 in
    column j % D only: the outputs are whole counts over whole counts, so
    one key too many or too few shows at any length."""
    rng = np.random.default_rng(3)
    P, H = 64, 1
    kv, ql = [a for a, _ in seqs], [b for _, b in seqs]
    pages = sum(-(-n // P) for n in kv) + 1
    table = ref.tables(rng, pages, kv, P)
    codes = rng.integers(0, 0x7f, (pages, 2, H, P, D)).astype(np.uint8)
    for b, n in enumerate(kv):
        for i in range(-(-n // P)):
            j = np.arange(i * P, (i + 1) * P)
            hot = np.zeros((P, D), np.uint8)
            hot[np.arange(P), j % D] = 0x38                     # 1.0
            hot[j >= n] = 0x7f                                  # what lies behind the sequence is NaN
            codes[table[b, i], 1, 0] = hot
            codes[table[b, i], 0, 0, j >= n] = 0x7f
    exps = np.zeros((pages, 2, H), np.int8)
    q = np.zeros((sum(ql), G, D), np.float16)
    got = attend_gpu(gpu, codes, exps, table, kv, ql, q, "f16", window=window, sinks=sinks)
    at = 0
    for n, m in zip(kv, ql):
        see = ref.sees(n, m, window, sinks).astype(float)
        count = np.zeros((m, D))
        np.add.at(count.T, np.arange(n) % D, see.T)
        want = count / see.sum(1, keepdims=True)
        # the counts are exact, 1 / l and the product round in f32, the output in f16
        tol = want * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25
        assert (np.abs(got[at:at + m].astype(float) - want[:, None]) <= tol[:, None]).all()
        at += m


@pytest.mark.parametrize("D,G,n", [(128, 8, 1), (64, 2, 3), (128, 4, 40)])
def test_nan_in_hidden_places_stays_there(gpu, D, G, n):
    """NaN keys and values outside a row's window, ahead of it or behind the
    sequence leave the row finite; the rows that see one are NaN."""
    rng = np.random.default_rng(5)
    P, L, window = 64, 300, 70
    pages = 7
    codes, exps = ref.pool(rng, pages, 1, P, D)
    table = ref.tables(rng, pages, [L], P)
    for j in (3, 100, L - n - window, L + 5):
        if j >= 0:
            codes[table[0, j // P], :, 0, j % P] = 0x7f
    codes[table[0, (L - 1) // P], 1, 0, (L - 1) % P, D // 2] = 0xff      # one value of the newest key
    q = rng.standard_normal((n, G, D)).astype(np.float16)
    got = attend_gpu(gpu, codes, exps, table, [L], [n], q, "f16", window=window)
    want, bound = ref.attend(codes, exps, table, [L], [n], q.astype(float), D ** -0.5, window)
    assert np.isnan(want).any() and not np.isnan(want).all()
    assert ref.close(got, want, bound, "f16")


@pytest.mark.parametrize("n", [1, 50])
def test_scales_far_apart(gpu, n):
    """Pages from one end of the exponents' range to the other, and queries
    of very unlike rows."""
    rng = np.random.default_rng(11)
    P, D, L, G = 64, 64, 64 * 6 + 9, 4
    codes, exps = ref.pool(rng, 8, 1, P, D, spread=0.0)
    table = ref.tables(rng, 8, [L], P)
    exps[:, 1, 0] = [-32, 63, 0, 40, -10, 5, -32, 20]
    exps[:, 0, 0] = [-20, -6, -10, -6, -7, -9, -6, -30]
    q = rng.standard_normal((n, G, D))
    q *= 10.0 ** np.array([-30, 0, 0.5, -3])[None, :, None]
    q = q.astype(ml_dtypes.bfloat16)
    got = attend_gpu(gpu, codes, exps, table, [L], [n], q, "bf16")
    want, bound = ref.attend(codes, exps, table, [L], [n], q.astype(float), D ** -0.5)
    assert np.isfinite(want).all() and ref.close(got, want, bound, "bf16")


def test_attend_strides_scale_and_layers(gpu):
    """q and out as slices of wider rows, another layer, a negative scale."""
    rng = np.random.default_rng(2)
    P, D, H, G, kv, ql = 64, 128, 2, 3, [140, 77], [1, 2]
    both = [ref.pool(rng, 6, H, P, D) for _ in range(2)]
    codes, exps = np.stack([a for a, _ in both]), np.stack([b for _, b in both])
    table = ref.tables(rng, 6, kv, P)
    cache, _, _ = cache_of(gpu, codes, exps)
    wide = rng.standard_normal((3, H * G + 4, D + 16)).astype(NP["bf16"])
    batch = cache.batch(table, kv, ql)
    from ptxgen import DeviceArray
    st = ((H * G + 4) * (D + 16), D + 16, 1)
    qd = gpu.put(wide, "bf16")
    q = DeviceArray(qd.ptr + 2 * (D + 16) * 2, "bf16", (3, H * G, D), st)      # heads 2 ..
    od = gpu.put(np.zeros_like(wide), "bf16")
    out = DeviceArray(od.ptr + 32, "bf16", (3, H * G, D), st)                  # columns 16 ..
    batch.attend(1, q, out, scale=-0.25)
    got = gpu.get(od, wide.shape, NP["bf16"])
    want, bound = ref.attend(codes[1], exps[1], table, kv, ql,
                             wide[:, 2:2 + H * G, :D].astype(float), -0.25)
    assert ref.close(got[:, :H * G, 16:], want, bound, "bf16")
    assert not got[:, H * G:].astype(float).any() and not got[..., :16].astype(float).any()
    batch.close()


APPENDS = [
    (128, 64, 2, "bf16", [(1, 1), (64, 64), (65, 65), (70, 6), (200, 130)]),
    (64, 64, 3, "f16", [(1, 1), (2, 1), (64, 1), (65, 1), (66, 1), (300, 1), (7, 0), (0, 0)]),
    (128, 128, 1, "f32", [(129, 2), (128, 100), (400, 272)]),
    (64, 256, 2, "bf16", [(600, 345), (256, 1), (257, 1)]),
    (128, 256, 1, "f16", [(256, 256), (300, 299)]),
    (64, 128, 1, "f32", [(1, 1), (130, 7)]),
]


@pytest.mark.parametrize("D,P,H,dtype,seqs", APPENDS)
def test_append(gpu, D, P, H, dtype, seqs):
    rng = np.random.default_rng(D + P)
    kv, ql = [a for a, _ in seqs], [b for _, b in seqs]
    pages = sum(-(-n // P) for n in kv) + 2
    codes, exps = ref.pool(rng, pages, H, P, D)
    table = ref.tables(rng, pages, kv, P)
    n = sum(ql)
    x = rng.standard_normal((2, n + 2, H, D)) * 2.0 ** rng.integers(-6, 7, (2, n + 2, H, 1))
    x = x.astype(NP[dtype])
    cache, cd, ed = cache_of(gpu, codes[None], exps[None])
    batch = cache.batch(table, kv, ql)
    batch.append(0, gpu.put(x[0], dtype), gpu.put(x[1], dtype))
    batch.check_errors()
    want = ref.append(codes, exps, table, kv, ql, x[0].astype(float), x[1].astype(float))
    assert (gpu.get(ed, exps.shape, np.int8) == want[1]).all()
    assert (gpu.get(cd, codes.shape, np.uint8) == want[0]).all()
    batch.close()


def test_append_values_at_the_edges(gpu):
    """Zeros, subnormals, 448 * 2^e and its neighbours, the range's ends,
    infinities and NaN; ties to even; strided keys and values."""
    D, P, H = 64, 64, 1
    rows = [np.zeros(D), np.full(D, 448.0), np.full(D, np.nextafter(np.float32(448), np.float32(449))),
            np.full(D, 1e-45), np.linspace(-1, 1, D), np.full(D, 3e38), np.full(D, 448 * 2.0 ** -32),
            np.r_[np.inf, -np.inf, np.nan, np.linspace(-3, 3, D - 3)], np.full(D, np.nan),
            np.r_[[17, 18, 19, 20, 21, 22, 23, 248, 264, 440, 448], np.full(D - 11, 2.0 ** -9 * 1.5)]]
    x = np.array(rows, np.float32)[:, None]                    # [10, 1, D]
    n = len(rows)
    codes = np.full((n, 2, H, P, D), 0x7f, np.uint8)
    exps = np.full((n, 2, H), 100, np.int8)                    # what a fresh page held does not matter
    table = np.arange(n, dtype=np.int32)[:, None]
    cache, cd, ed = cache_of(gpu, codes[None], exps[None])
    batch = cache.batch(table, [1] * n)
    wide = np.zeros((n, 3, H, D + 4), np.float32)
    wide[:, 1, :, 4:], wide[:, 2, :, 4:] = x, -x
    from ptxgen import DeviceArray
    w = gpu.put(wide, "f32")
    st = (3 * H * (D + 4), D + 4, 1)
    k = DeviceArray(w.ptr + 4 * (H * (D + 4) + 4), "f32", (n, H, D), st)
    v = DeviceArray(w.ptr + 4 * (2 * H * (D + 4) + 4), "f32", (n, H, D), st)
    batch.append(0, k, v)
    want = ref.append(codes, exps, table, [1] * n, [1] * n, x.astype(float), -x.astype(float))
    got = gpu.get(cd, codes.shape, np.uint8)
    assert (gpu.get(ed, exps.shape, np.int8) == want[1]).all()
    nan = np.isnan(ref.DECODE[want[0]])
    assert (got == want[0])[~nan].all() and np.isnan(ref.DECODE[got[nan]]).all()
    batch.close()


@pytest.mark.parametrize("layers,pages,H,P,D,n", [(3, 9, 1, 64, 64, 4), (2, 40, 3, 128, 128, 17),
                                                  (1, 1100, 1, 64, 64, 520)])
def test_copy_pages(gpu, layers, pages, H, P, D, n):
    rng = np.random.default_rng(pages)
    codes = rng.integers(0, 256, (layers, pages, 2, H, P, D)).astype(np.uint8)
    exps = rng.integers(-32, 64, (layers, pages, 2, H)).astype(np.int8)
    order = rng.permutation(pages)
    src, dst = order[:n].copy(), order[n:2 * n]
    src[-1] = src[0]                                           # a page may be copied twice
    cache, cd, ed = cache_of(gpu, codes, exps)
    cache.copy_pages(src.tolist(), dst.tolist())
    codes[:, dst], exps[:, dst] = codes[:, src], exps[:, src]
    assert (gpu.get(cd, codes.shape, np.uint8) == codes).all()
    assert (gpu.get(ed, exps.shape, np.int8) == exps).all()


def test_bad_tables_on_the_device_are_reported(gpu):
    """A captured call reads its table on the device: a page outside the pool
    hides its keys, lengths that cannot be right skip the sequence; both
    are reported and touch nothing else."""
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(8)
    P, D, kv = 64, 64, [130, 70, 40]
    codes, exps = ref.pool(rng, 8, 1, P, D)
    table = ref.tables(rng, 8, kv, P)
    cache, cd, _ = cache_of(gpu, codes[None], exps[None])
    q = rng.standard_normal((3, 2, D)).astype(np.float16)
    batch = cache.batch(table, kv)
    qd, od = gpu.put(q, "f16"), gpu.put(np.full_like(q, 77.0), "f16")
    bad = table.copy()
    bad[0, 1] = 8                                              # one past the pool
    gpu.dev.htod(batch._d.page_table, bad)
    gpu.dev.htod(batch._d.kv_lens + 4, np.array([1000], np.int32))
    batch.attend(0, qd, od)
    with pytest.raises(EmmyError, match="0x40"):
        batch.check_errors()
    batch.check_errors()                                       # cleared
    got = gpu.get(od, q.shape, np.float16)
    assert (got[1] == 77.0).all()
    see = np.r_[0:64, 128:130]                                 # the keys of the two good pages
    k, v = ref.held(codes, exps, table, 0, 130, 0)
    for g in range(2):
        s = q[0, g].astype(float) @ k[see].T / 8
        p = np.exp(s - s.max())
        assert np.abs(p @ v[see] / p.sum() - got[0, g].astype(float)).max() < 0.02 * np.abs(v[see]).max()
    k = rng.standard_normal((3, 1, D)).astype(np.float16)
    bad[0, 2] = -1
    gpu.dev.htod(batch._d.page_table, bad)
    before = gpu.get(cd, codes.shape, np.uint8)
    batch.append(0, gpu.put(k, "f16"), gpu.put(k, "f16"))
    with pytest.raises(EmmyError, match="0x40"):
        batch.check_errors()
    after = gpu.get(cd, codes.shape, np.uint8)
    changed = {int(p) for p in np.nonzero((before != after).any((1, 2, 3, 4)))[0]}
    assert changed <= {int(table[2, 0])}
    batch.close()


def test_decoding_run(gpu):
    """Prompts, single tokens, a fork that diverges, rejected drafts, a freed
    sequence and a compaction, against the same run on the host."""
    from ptxgen import KVCache, KVSequences
    rng = np.random.default_rng(21)
    P, D, H, G, layers, pages = 64, 64, 2, 2, 2, 24
    cache = KVCache(pages, H, D, layers=layers)
    seqs = KVSequences(cache)
    codes = np.zeros((layers, pages, 2, H, P, D), np.uint8)
    exps = np.zeros((layers, pages, 2, H), np.int8)

    def step(sids, q_lens):
        held = [seqs.pages(s) for s in sids]
        batch = seqs.batch(sids, q_lens)
        table, kv = seqs.table(sids), [seqs.length(s) for s in sids]
        for s, old in zip(sids, held):                         # pages copied on write
            for a, b in zip(old, seqs.pages(s)):
                if a != b:
                    codes[:, b], exps[:, b] = codes[:, a], exps[:, a]
        n = sum(q_lens)
        for layer in range(layers):
            k, v = (rng.standard_normal((2, n, H, D)) * 2.0 ** rng.integers(-2, 3)).astype(np.float16)
            q = rng.standard_normal((n, H * G, D)).astype(np.float16)
            batch.append(layer, gpu.put(k, "f16"), gpu.put(v, "f16"))
            out = gpu.put(np.zeros_like(q), "f16")
            batch.attend(layer, gpu.put(q, "f16"), out)
            codes[layer], exps[layer] = ref.append(codes[layer], exps[layer], table, kv, q_lens,
                                                   k.astype(float), v.astype(float))
            want, bound = ref.attend(codes[layer], exps[layer], table, kv, q_lens, q.astype(float), D ** -0.5)
            assert ref.close(gpu.get(out, q.shape, np.float16), want, bound, "f16")
        batch.check_errors()
        return batch

    a, b = seqs.new(), seqs.new()
    step([a, b], [100, 30])
    for _ in range(3):
        step([a, b], [1, 1])
    c = seqs.fork(a)
    d = seqs.fork(a)
    step([a, b, c, d], [1, 5, 1, 2])
    assert len({seqs.pages(s)[1] for s in (a, c, d)}) == 3 and seqs.pages(a)[0] == seqs.pages(c)[0]
    seqs.truncate(b, 34)
    step([b, c], [3, 70])
    seqs.free(a)
    old = step([b, d], [1, 1])
    where = {s: seqs.pages(s) for s in (b, c, d)}
    used = seqs.compact()
    assert max(max(seqs.pages(s)) for s in (b, c, d)) < used == pages - seqs.free_pages
    moved_c, moved_e = codes.copy(), exps.copy()
    for s, pg in where.items():
        for x, y in zip(pg, seqs.pages(s)):
            moved_c[:, y], moved_e[:, y] = codes[:, x], exps[:, x]
    codes, exps = moved_c, moved_e
    from ptxgen.runtime import EmmyError
    with pytest.raises(EmmyError, match="compact"):
        old.append(0, gpu.put(np.zeros((2, H, D), np.float16), "f16"), gpu.put(np.zeros((2, H, D), np.float16), "f16"))
    step([d, b, c], [1, 1, 64])
    cache.close()
