"""The paged 8-bit cache on the CPU: what its calls refuse, the page
bookkeeping against a model, and the oracle's e4m3 against ml_dtypes."""

import ctypes as C
import random

import ml_dtypes
import numpy as np
import pytest

from ptxgen import kvcache as kv
from ptxgen.kvcache import DeviceArray, KVCache, KVSequences
from ptxgen.runtime import EmmyError
from tests import kv8_oracle as ref


class FakeLib:
    """Every entry point succeeds and is noted."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*a):
            self.calls.append((name, a))
            if name == "emmy_kv8_attend_sizes":
                a[2]._obj.value, a[3]._obj.value = 5000, 3000
            return 0
        return call


class FakeDevice:
    def __init__(self, lib):
        self.L, self.stream, self.next = lib, C.c_void_p(7), 4096
        self.live = set()

    def alloc(self, n):
        self.next += (n + 4095) // 4096 * 4096
        self.live.add(self.next)
        return self.next

    def free(self, p):
        self.live.remove(p)

    def memset32(self, *a):
        pass

    def event(self):
        return 99

    def sync(self, *a):
        pass


@pytest.fixture
def dev(monkeypatch):
    lib = FakeLib()
    d = FakeDevice(lib)
    monkeypatch.setattr(kv, "load_library", lambda: lib)
    monkeypatch.setattr(kv.Device, "get", classmethod(lambda cls, ordinal=0: d))
    return d


def small(dev, **kw):
    return KVCache(**{"pages": 10, "kv_heads": 2, "head_dim": 64, "layers": 3, **kw})


@pytest.mark.parametrize("kw,says", [
    ({"head_dim": 96}, "head_dim"), ({"page_size": 48}, "page_size"), ({"page_size": 16}, "page_size"),
    ({"kv_heads": 0}, "kv_heads"), ({"pages": 0}, "pages"), ({"layers": 0}, "layers"),
])
def test_cache_refusals(dev, kw, says):
    with pytest.raises(EmmyError, match=says):
        small(dev, **kw)


@pytest.mark.parametrize("codes,exps,says", [
    (("u8", (3, 10, 2, 2, 64, 65)), ("i8", (3, 10, 2, 2)), "shape"),
    (("u8", (3, 10, 2, 2, 64, 64)), ("i8", (3, 10, 2)), "shape"),
    (("f16", (3, 10, 2, 2, 64, 64)), ("i8", (3, 10, 2, 2)), "8-bit"),
    (("u8", (3, 10, 2, 2, 64, 64)), ("u8", (3, 10, 2, 2)), "8-bit"),
    (("u8", (3, 10, 2, 2, 64, 64), (2, 1, 1, 1, 1, 1)), ("i8", (3, 10, 2, 2)), "contiguous"),
    (("u8", (3, 10, 2, 2, 64, 64), None, 1), ("i8", (3, 10, 2, 2)), "device"),
])
def test_storage_refusals(dev, codes, exps, says):
    with pytest.raises(EmmyError, match=says):
        small(dev, storage=(DeviceArray(4096, *codes), DeviceArray(8192, *exps)))
    with pytest.raises(EmmyError, match="aligned"):
        small(dev, storage=(DeviceArray(4100, "u8", (3, 10, 2, 2, 64, 64)),
                            DeviceArray(8192, "i8", (3, 10, 2, 2))))


@pytest.mark.parametrize("table,lens,q,says", [
    ([1, 2], [3], None, "page_table"), ([[]], [0], None, "page_table"),
    ([[1.5]], [1], None, "whole"), ([[1], [2]], [1], None, "lengths"),
    ([[1]], [1], [1, 1], "lengths"), ([[1]], [0], None, "new tokens"),
    ([[1]], [5], [6], "new tokens"), ([[1]], [5], [-1], "new tokens"),
    ([[1]], [65], None, "longer"), ([[1, 10]], [65], None, "outside"),
    ([[-1]], [3], None, "outside"), ([[0]] * 4097, [1] * 4097, None, "at most"),
    ([[0] * (2 ** 24 + 1)], [1], None, "2\\^30"),
])
def test_batch_refusals(dev, table, lens, q, says):
    with pytest.raises(EmmyError, match=says):
        small(dev).batch(table, lens, q)


def test_unused_table_entries_do_not_matter(dev):
    small(dev).batch([[3, 99, -7], [1, 2, 999]], [64, 128])


def test_call_refusals(dev):
    cache = small(dev)
    b = cache.batch([[1], [2]], [5, 6], [1, 2])
    q = DeviceArray(1 << 20, "bf16", (3, 4, 64))
    out = DeviceArray(1 << 21, "bf16", (3, 4, 64))
    k = DeviceArray(1 << 22, "f32", (3, 2, 64))
    assert b.attend(2, q, out) is out
    b.append(0, k, k)
    bad = [
        (lambda: b.attend(3, q, out), "layer 3"), (lambda: b.append(-1, k, k), "layer -1"),
        (lambda: b.attend(0, DeviceArray(1, "bf16", (2, 4, 64)), out), "q has shape"),
        (lambda: b.attend(0, DeviceArray(1, "bf16", (3, 4, 128)), out), "q has shape"),
        (lambda: b.attend(0, DeviceArray(1, "bf16", (12, 64)), out), "q has shape"),
        (lambda: b.attend(0, q, DeviceArray(1, "bf16", (3, 2, 64))), "out has shape"),
        (lambda: b.attend(0, q, DeviceArray(1, "f16", (3, 4, 64))), "both"),
        (lambda: b.attend(0, k, k), "bf16 or f16"),
        (lambda: b.attend(0, DeviceArray(1, "f64", (3, 4, 64)), out), "dtype"),
        (lambda: b.attend(0, DeviceArray(1, "bf16", (3, 4, 64), (512, 128, 2)), out), "contiguous"),
        (lambda: b.attend(0, DeviceArray(1, "bf16", (3, 4, 64), None, 1), out), "device"),
        (lambda: b.append(0, k, DeviceArray(1, "bf16", (3, 2, 64))), "both"),
        (lambda: b.append(0, DeviceArray(1, "f32", (3, 4, 64)), k), "k has shape"),
        (lambda: b.append(0, DeviceArray(1, "u8", (3, 2, 64)), DeviceArray(1, "u8", (3, 2, 64))), "both"),
        (lambda: b.attend(0, q, out, window=2 ** 32 + 5), "window"),
        (lambda: b.attend(0, q, out, window=-1), "window"),
        (lambda: b.attend(0, q, out, window=1, sinks=2 ** 31), "sinks"),
        (lambda: b.update([[1], [2]], [5, 6], [2, 2]), "made for"),
        (lambda: b.update([[1, 2], [2, 3]], [5, 6], [1, 2]), "table"),
    ]
    for call, says in bad:
        with pytest.raises(EmmyError, match=says):
            call()
    clash = cache.batch([[1], [1]], [5, 6])
    clash.attend(0, DeviceArray(1 << 20, "bf16", (2, 4, 64)), DeviceArray(1 << 21, "bf16", (2, 4, 64)))
    with pytest.raises(EmmyError, match="same page"):
        clash.append(0, k, k)
    b.close()
    with pytest.raises(EmmyError, match="closed"):
        b.attend(0, q, out)
    cache.close()
    for call in (lambda: clash.attend(0, q, out), lambda: cache.copy_pages([1], [2])):
        with pytest.raises(EmmyError, match="cache is closed"):
            call()


def test_another_stream_waits_for_the_batch_once(dev):
    b = small(dev).batch([[1]], [9], stream=5)
    q, out = DeviceArray(1 << 20, "bf16", (1, 4, 64)), DeviceArray(1 << 21, "bf16", (1, 4, 64))
    dev.L.calls.clear()
    for st in (5, 6, 6, 0, 6):
        b.attend(0, q, out, stream=st)
    waits = [a[0] for name, a in dev.L.calls if name == "emmy_stream_wait_event"]
    assert waits == [6, 0]
    zeroed = [a[3] for name, a in dev.L.calls if name == "emmy_memset_d32"]
    assert zeroed == [5]                         # the workspace, on the stream that needed it


def test_one_plan_for_each_heads_window_and_sinks(dev):
    """Made once, made again by update, and allocated before a capture by
    reserve."""
    b = small(dev).batch([[1]], [9])
    q, out = DeviceArray(1 << 20, "bf16", (1, 4, 64)), DeviceArray(1 << 21, "bf16", (1, 4, 64))

    def plans():
        n = sum(name == "emmy_kv8_attend_plan" for name, _ in dev.L.calls)
        dev.L.calls.clear()
        return n
    for layer in range(3):
        b.attend(layer, q, out)
    assert plans() == 1
    b.reserve(4, 100, 4)
    assert plans() == 1
    live = set(dev.live)
    b.attend(0, q, out, window=100, sinks=4)
    assert plans() == 0 and dev.live == live
    b.update([[1]], [10])
    assert plans() == 2 and dev.live == live


def test_closed_batches_give_their_buffers_to_the_next_on_their_stream(dev):
    cache = small(dev)
    q, out = DeviceArray(1 << 20, "bf16", (1, 4, 64)), DeviceArray(1 << 21, "bf16", (1, 4, 64))

    def run(made_on, used_on):
        b = cache.batch([[1]], [9], stream=made_on)
        b.attend(0, q, out, stream=used_on)
        held = {p for p, _ in b._held}
        b.close()
        return held
    first = run(1, 1)
    assert run(1, 1) == first                    # no wait is needed
    assert not run(2, 2) & first                 # another stream
    assert not run(1, 2) & dev.live              # used on two: freed, which waits
    other = small(dev)                           # another cache of the device
    cache, second = other, run(2, 2)
    assert run(2, 2) == second
    storage = {other.codes, other.exps}
    other.close()
    assert not storage & dev.live and second <= dev.live


def test_spare_buffers_are_bounded(dev, monkeypatch):
    monkeypatch.setattr(kv._Pool, "MOST", 8192)
    cache = small(dev)
    batches = [cache.batch([[1]], [9], stream=1) for _ in range(5)]
    for b in batches:
        b.close()
    assert len(dev._kv_pool.held["batch", 4096, 1]) == 2
    assert dev._kv_pool.bytes == 8192 and len(dev.live - set(cache._own)) == 2


def test_stream_arguments(dev):
    """None is the device's stream, 0 the legacy default stream."""
    class Torchlike:
        cuda_stream = 33
    assert [kv._stream_of(s, dev) for s in (None, 0, 5, Torchlike(), C.c_void_p(9), C.c_void_p(0))] \
        == [7, 0, 5, 33, 9, 0]


@pytest.mark.parametrize("src,dst,says", [
    ([1], [2, 3], "same length"), ([10], [2], "outside"), ([1], [-1], "outside"),
    ([1, 2], [3, 3], "twice"), ([1, 2], [2, 3], "both"), ([1.5], [2], "page numbers"),
    ([1], [2 ** 40], "page numbers"),
])
def test_copy_refusals(dev, src, dst, says):
    cache = small(dev)
    cache.copy_pages([], [])
    cache.copy_pages([1, 1], np.array([2, 3]))
    with pytest.raises(EmmyError, match=says):
        cache.copy_pages(src, dst)


def test_long_copy_lists_are_cut(dev):
    cache = small(dev, pages=3000)
    cache.copy_pages(list(range(1000)), list(range(1000, 2000)))
    counts = [a[4] for name, a in dev.L.calls if name == "emmy_kv8_copy_pages"]
    assert sum(counts) == 1000 and max(counts) <= kv.MAX_PAIRS


class ModelCache(KVCache):
    """Pages as lists of token values; copies are made on the host."""

    def copy_pages(self, src, dst, stream=None):
        super().copy_pages(src, dst, stream)
        for a, b in zip(src, dst):
            self.content[b] = list(self.content[a])


@pytest.mark.parametrize("seed", range(6))
def test_sequences_against_a_model(dev, seed):
    """Random appends, forks, truncations, frees and compactions: every
    sequence keeps its own tokens, whatever shares its pages."""
    rng = random.Random(seed)
    cache = ModelCache(pages=24, kv_heads=1, head_dim=64)
    cache.content = {p: [None] * 64 for p in range(24)}
    seqs = KVSequences(cache)
    want: dict[int, list] = {}
    token = refused = 0
    for _ in range(400):
        live = list(want)
        do = rng.random()
        if not live or do < 0.1:
            want[seqs.new()] = []
        elif do < 0.6:
            some = rng.sample(live, rng.randint(1, len(live)))
            q = [rng.choice([0, 1, 1, 5, 64, 100]) for _ in some]
            before = ({s: seqs.pages(s) for s in live}, seqs.free_pages, list(seqs._refs))
            try:
                batch = seqs.batch(some, q)
            except EmmyError as exc:
                assert "pages needed" in str(exc)
                refused += 1
                assert before == ({s: seqs.pages(s) for s in live}, seqs.free_pages, list(seqs._refs))
                assert all(seqs.length(s) == len(want[s]) for s in live)
                continue
            assert not batch._clash
            for s, n in zip(some, q):
                for _ in range(n):
                    at = len(want[s])
                    page = seqs.pages(s)[at // 64]
                    assert seqs._refs[page] == 1
                    cache.content[page][at % 64] = token
                    want[s].append(token)
                    token += 1
        elif do < 0.75:
            s = rng.choice(live)
            want[seqs.fork(s)] = list(want[s])
        elif do < 0.87:
            s = rng.choice(live)
            n = rng.randint(0, len(want[s]))
            seqs.truncate(s, n)
            del want[s][n:]
        elif do < 0.95:
            s = rng.choice(live)
            seqs.free(s)
            del want[s]
        else:
            used = seqs.compact()
            assert all(p < used for s in want for p in seqs.pages(s))
            assert used == 24 - seqs.free_pages
        for s, tokens in want.items():
            assert seqs.length(s) == len(tokens) and len(seqs.pages(s)) == -(-len(tokens) // 64)
            got = [cache.content[seqs.pages(s)[i // 64]][i % 64] for i in range(len(tokens))]
            assert got == tokens
        used = {p for s in want for p in seqs.pages(s)}
        assert len(used) + seqs.free_pages == 24 and len(set(seqs._free)) == seqs.free_pages
        assert not used & set(seqs._free)
    assert refused


def test_sequence_refusals(dev):
    cache = small(dev)
    seqs = KVSequences(cache)
    a = seqs.new()
    for call, says in [(lambda: seqs.length(9), "no sequence"), (lambda: seqs.fork(9), "no sequence"),
                       (lambda: seqs.truncate(a, 1), "0 tokens"), (lambda: seqs.batch([]), "at least one"),
                       (lambda: seqs.batch([a, a]), "twice"), (lambda: seqs.batch([a], [-1]), "negative"),
                       (lambda: seqs.batch([a], [1, 2]), "q_len"), (lambda: seqs.batch([a], [641]), "11 pages"),
                       (lambda: seqs.batch([9]), "no sequence")]:
        with pytest.raises(EmmyError, match=says):
            call()
    assert seqs.free_pages == 10
    b = seqs.batch([a], [65])
    c = seqs.new()
    seqs.batch([c])
    seqs.free(c)
    seqs.compact()
    assert not b._stale                          # nothing had to move
    c, d = seqs.new(), seqs.new()
    seqs.batch([c, d])
    seqs.free(c)
    old = seqs.batch([d])
    seqs.compact()
    with pytest.raises(EmmyError, match="compact"):
        old.append(0, DeviceArray(16, "f32", (1, 2, 64)), DeviceArray(16, "f32", (1, 2, 64)))
    old.update(seqs.table([d]), [seqs.length(d)])
    old.append(0, DeviceArray(16, "f32", (1, 2, 64)), DeviceArray(16, "f32", (1, 2, 64)))


def test_a_batch_that_cannot_be_made_leaves_the_books(dev, monkeypatch):
    """Too many sequences, a copy that fails, a closed cache: pages, lengths
    and reference counts stay as they were."""
    cache = KVCache(pages=5000, kv_heads=2, head_dim=64)
    seqs = KVSequences(cache)
    a = seqs.new()
    seqs.batch([a], [70])
    many = [a, seqs.fork(a)] + [seqs.new() for _ in range(4095)]

    def books():
        return ({s: seqs.pages(s) for s in many}, [seqs.length(s) for s in many], list(seqs._refs), list(seqs._free))
    before = books()
    with pytest.raises(EmmyError, match="4096"):
        seqs.batch(many)
    assert books() == before
    with monkeypatch.context() as m:
        m.setattr(kv, "_copy_in", lambda *a: kv.check(-3, "htod"))
        with pytest.raises(EmmyError):
            seqs.batch(many[:9], [100] * 9)
    assert books() == before
    cache.close()
    with pytest.raises(EmmyError, match="closed"):
        seqs.batch(many[:2])                     # one of them has to copy
    assert books() == before
    with pytest.raises(EmmyError, match="no sequence"):
        seqs.table([a, 99999])


def test_host_copies_are_refused_while_a_stream_is_captured(dev):
    """Making, updating, planning and checking a batch; a refused update keeps
    what append knows of the batch's pages."""
    cache = small(dev)
    b = cache.batch([[1], [2]], [9, 9], stream=5)
    dev.L.emmy_stream_capturing = lambda st, word: setattr(word._obj, "value", 1) or 0
    for call in (lambda: cache.batch([[1]], [9], stream=5), lambda: b.update([[1], [1]], [9, 9], stream=5),
                 lambda: b.reserve(4, stream=5), lambda: b.check_errors(stream=5)):
        with pytest.raises(EmmyError, match="captured"):
            call()
    x = DeviceArray(1 << 20, "bf16", (2, 2, 64))
    b.append(0, x, x, stream=5)                  # the pages are still two
    with pytest.raises(EmmyError):
        b.update([[1], [99]], [9, 9])
    b.append(0, x, x, stream=5)


def _library():
    from ptxgen.runtime import lib_path, load_library
    if not lib_path().exists():
        import subprocess
        from pathlib import Path
        subprocess.run(["make", "-C", str(Path(__file__).resolve().parent.parent / "emmy-ptx_b200")], check=True)
    return load_library()


def _desc(**kw):
    d = kv._Cache()
    for k, v in {**dict(codes=4096, exps=4096, page_table=4096, kv_lens=4096, q_starts=4096, pages=8,
                        kv_heads=2, head_dim=64, page_size=64, seqs=1, table_width=2, tokens=3, max_q=3),
                 **kw}.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,says", [
    ({"codes": 0}, "null cache storage"), ({"codes": 4104}, "16-byte"), ({"head_dim": 80}, "head_dim"),
    ({"page_size": 32}, "page_size"), ({"kv_heads": 0}, "kv_heads"), ({"pages": 0}, "no pages"),
    ({"device": -1}, "device"), ({"page_table": 0}, "null page table"), ({"kv_lens": 4098}, "4-byte"),
    ({"seqs": 0}, "seqs"), ({"seqs": 4097}, "seqs"), ({"table_width": 0}, "table_width"),
    ({"max_q": 4}, "max_q"), ({"table_width": 2 ** 25}, "2\\^30"),
])
def test_c_entry_points_refuse_bad_descriptions(kw, says):
    L = _library()
    d = _desc(**kw)
    st = (C.c_int64 * 2)(128, 64)
    assert L.emmy_kv8_append(C.byref(d), 4096, 4096, 0, st, st, None) == -3
    with pytest.raises(EmmyError, match=says):
        kv.check(-3)
    a = kv._Attend(heads=4, plan=4096, plan_bytes=1 << 30)
    assert L.emmy_kv8_attend(C.byref(d), C.byref(a), None) == -3


def test_c_entry_points_refuse_bad_arguments():
    L = _library()
    d = _desc()
    st, odd = (C.c_int64 * 2)(128, 64), (C.c_int64 * 2)(129, 64)
    for args, says in [((4096, 4096, 3, st, st), "dtype"), ((0, 4096, 1, st, st), "null k or v"),
                       ((4096, 4104, 1, st, st), "16 bytes"), ((4096, 4096, 1, odd, st), "16 bytes"),
                       ((4096, 4096, 0, st, None), "null strides")]:
        assert L.emmy_kv8_append(C.byref(d), *args, None) == -3
        with pytest.raises(EmmyError, match=says):
            kv.check(-3)
    assert L.emmy_kv8_append(C.byref(_desc(tokens=0, max_q=0)), 0, 0, 1, st, st, None) == 0
    assert L.emmy_kv8_append(None, 0, 0, 1, st, st, None) == -3
    one = (C.c_int32 * 1)(3)
    for args, says in [((0, one, one, 1), "layers"), ((1, one, one, 481), "480"),
                       ((1, None, one, 1), "null"), ((1, one, (C.c_int32 * 1)(8), 1), "outside"),
                       ((1, (C.c_int32 * 1)(-1), one, 1), "outside")]:
        assert L.emmy_kv8_copy_pages(C.byref(d), *args, None) == -3
        with pytest.raises(EmmyError, match=says):
            kv.check(-3)
    assert L.emmy_kv8_copy_pages(C.byref(d), 1, None, None, 0, None) == 0
    u = C.c_uint64()
    assert L.emmy_kv8_attend_sizes(C.byref(d), 3, C.byref(u), C.byref(u)) == -3     # not a multiple
    assert L.emmy_kv8_attend_sizes(C.byref(d), 4, None, C.byref(u)) == -3
    assert L.emmy_kv8_attend_plan(C.byref(d), None, None) == -3
    for kw in ({"seqs": -1}, {"tokens": -4, "max_q": -4}, {"max_q": 9}, {"table_width": 0}):
        assert L.emmy_kv8_attend_sizes(C.byref(_desc(**kw)), 4, C.byref(u), C.byref(u)) == -3


def test_oracle_rounds_as_e4m3_does():
    rng = np.random.default_rng(0)
    x = np.r_[rng.standard_normal(20000) * 2.0 ** rng.integers(-12, 9, 20000), ref.DECODE[:127],
              (ref.DECODE[:126] + ref.DECODE[1:127]) / 2].astype(np.float32)
    x = np.r_[x, -x]
    x = x[np.abs(x) <= 448]
    want = x.astype(ml_dtypes.float8_e4m3fn).view(np.uint8)
    assert (ref.encode(x) == want).all()
    codes = np.arange(256, dtype=np.uint8)
    ours, theirs = ref.DECODE, codes.view(ml_dtypes.float8_e4m3fn).astype(np.float64)
    assert (np.isnan(ours) == np.isnan(theirs)).all() and (ours == theirs)[~np.isnan(ours)].all()
    assert [ref.exponent(a) for a in (0, 448, 449, 448 * 2.0 ** -32, 1e30)] == [-32, 0, 1, -32, 63]
