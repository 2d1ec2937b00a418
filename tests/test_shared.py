"""Shared prefixes on the CPU: which runs a batch finds, what it hands on, and
what the library refuses."""

import ctypes as C
import random

import numpy as np
import pytest

from ptxgen import kvcache as kv
from ptxgen.kvcache import DeviceArray, KVSequences
from tests.test_kvcache import dev, small  # noqa: F401 - a fixture


@pytest.fixture(autouse=True)
def share_all(monkeypatch):
    monkeypatch.setattr(kv, "MIN_SAVED", {64: 0, 128: 0})


def check(runs, alike):
    """Runs do not overlap, and share what all their sequences have in common."""
    end = 0
    for first, count, pages in runs:
        assert first >= end and count >= 2
        assert pages == min(alike[first:first + count - 1]) > 0
        end = first + count
    assert end <= len(alike) + 1


@pytest.mark.parametrize("alike,want", [
    ([3], [(0, 2, 3)]), ([3, 3, 3], [(0, 4, 3)]), ([1, 9], [(1, 2, 9)]), ([5, 4], [(0, 3, 4)]),
    ([7, 1, 1, 1], [(0, 2, 7), (2, 3, 1)]), ([2, 8, 8, 2], [(1, 3, 8)]), ([8, 8, 7, 8, 8], [(0, 6, 7)]),
    ([9, 9, 1, 9, 9], [(0, 3, 9), (3, 3, 9)]),
])
def test_best_runs(alike, want):
    assert kv._best_runs(alike) == want


def test_best_runs_hold():
    rng = random.Random(1)
    for _ in range(500):
        alike = [rng.randint(1, rng.choice([1, 3, 9])) for _ in range(rng.randint(1, 30))]
        runs = kv._best_runs(alike)
        check(runs, alike)
        # never fewer page reads saved than by one run of all, or by the best pair
        saved = sum((n - 1) * p for _, n, p in runs)
        assert saved >= max(len(alike) * min(alike), max(alike))
    assert kv._best_runs([4] * 4095) == [(0, 4096, 4)]
    check(kv._best_runs(list(range(1, 2000))), list(range(1, 2000)))
    check(kv._best_runs(list(range(2000, 0, -1))), list(range(2000, 0, -1)))


@pytest.mark.parametrize("table,lens,q,want", [
    # whole pages before any new token only
    ([[1, 2, 3], [1, 2, 4]], [130, 131], [1, 1], [(0, 2, 2)]),
    ([[1, 2, 3], [1, 2, 4]], [130, 131], [3, 1], [(0, 2, 1)]),
    ([[1, 2, 3], [1, 2, 4]], [130, 131], [130, 1], []),
    ([[1, 2], [1, 2]], [128, 128], [0, 0], [(0, 2, 2)]),
    ([[1, 2], [3, 2]], [100, 100], [1, 1], []),
    # what lies behind a sequence's last page does not count
    ([[1, 0, 0], [1, 0, 0]], [65, 70], [1, 1], [(0, 2, 1)]),
    # those that follow one another
    ([[1, 5], [1, 6], [2, 7], [1, 8], [1, 9]], [65, 66, 67, 68, 69], [1] * 5, [(0, 2, 1), (3, 2, 1)]),
    ([[3]], [60], [1], []),
])
def test_runs_of(table, lens, q, want):
    assert kv._runs_of(np.array(table), np.array(lens), np.array(q), 64) == want




def test_batch_hands_on(dev, monkeypatch):  # noqa: F811
    copies = []
    monkeypatch.setattr(kv, "_copy_in", lambda d, dst, host, st: copies.append((dst, host.copy())))
    cache = small(dev)
    table = [[1, 2, 3], [1, 2, 4], [1, 2, 5], [9, 0, 0]]
    batch = cache.batch(table, [130, 140, 129, 5], [1, 2, 1, 1], stream=3, shared=True)
    (dst, host), = copies
    assert host[-12:].reshape(3, 4).tolist() == [[0, 0, 0, 3], [3, 1, 1, 1], [128, 128, 128, 0]]
    assert batch._s.runs == dst + 4 * (len(host) - 12) and (batch._s.max_runs, batch._s.max_tokens) == (1, 4)
    q = DeviceArray(4096, "f16", (5, 4, 64))
    monkeypatch.setattr(dev.L, "emmy_kv8_attend_shared_sizes", lambda *a: setattr(a[3]._obj, "value", 5000) or setattr(a[4]._obj, "value", 300) or 0, raising=False)
    batch.attend(0, q, DeviceArray(8192, "f16", (5, 4, 64)), stream=3)
    names = [n for n, _ in dev.L.calls]
    assert "emmy_kv8_attend_shared_plan" in names and names[-1] == "emmy_kv8_attend_shared"
    assert "emmy_kv8_attend" not in names and dev.L.calls[-1][1][1] is batch._sref
    # an update with more: another run is left out, one of more tokens is split
    batch.update([[1, 2, 3], [1, 2, 4], [9, 2, 5], [9, 2, 6]], [130, 140, 65, 66], [1, 1, 1, 1], stream=3)
    runs = copies[-1][1][-12:].reshape(3, 4)
    assert runs.tolist() == [[0, 0, 2, 3], [2, 1, 1, 1], [128, 128, 0, 0]]
    batch.update([[1, 2, 3]] * 4, [130, 129, 129, 129], [2, 1, 1, 1], stream=3)
    runs = copies[-1][1][-12:].reshape(3, 4)
    assert runs.tolist() == [[0, 0, 0, 3], [3, 1, 1, 1], [128, 128, 128, 0]]


def test_batch_without_runs_is_as_ever(dev):  # noqa: F811
    for shared in (False, True):
        batch = small(dev).batch([[1], [2]], [9, 9], stream=3, shared=shared)
        assert batch._s is None
        batch.attend(0, DeviceArray(4096, "f16", (2, 4, 64)), DeviceArray(8192, "f16", (2, 4, 64)), stream=3)
    assert not any("shared" in n for n, _ in dev.L.calls)


@pytest.mark.parametrize("d,seqs,pages,shares", [(128, 16, 34, True), (128, 16, 33, False), (64, 11, 300, True),
                                                 (64, 11, 299, False), (128, 2, 500, True), (128, 1, 999, False)])
def test_little_is_not_shared(dev, monkeypatch, d, seqs, pages, shares):  # noqa: F811
    """(sequences - 1) * pages * kv heads reads saved, against what it costs."""
    monkeypatch.setattr(kv, "MIN_SAVED", {64: 6000, 128: 4000})
    heads = 8 if d == 128 and seqs > 2 else 2 if d == 64 else 8
    cache = small(dev, pages=4000, kv_heads=heads, head_dim=d)
    table = np.concatenate([np.tile(np.arange(pages), (seqs, 1)), 1000 + np.arange(seqs)[:, None]], 1)
    batch = cache.batch(table, [64 * pages + 1] * seqs, stream=3, shared=True)
    assert (batch._s is not None) == shares
    if shares:      # what it was made for stays, however little an update saves
        batch.update(table, [65] * seqs, stream=3)
        assert batch._s.max_runs == 1


@pytest.mark.parametrize("alone,long,shares", [(0, 1, True), (50, 1, True), (1000, 1, False), (50, 200, False)])
def test_sharing_pays_for_other_sequences(dev, monkeypatch, alone, long, shares):  # noqa: F811
    """8 sequences with 80 pages in common (4480 reads saved), beside others of so
    many pages of their own, whose rows and keys cost more in a batch that shares."""
    monkeypatch.setattr(kv, "MIN_SAVED", {64: 6000, 128: 4000})
    cache = small(dev, pages=20000, kv_heads=8, head_dim=128)
    table = np.zeros((8 + alone, 200), np.int32)
    table[:8, :80], table[:8, 80] = np.arange(80), 100 + np.arange(8)
    table[8:, :long] = 200 + np.arange(alone * long).reshape(alone, long)
    batch = cache.batch(table, [64 * 80 + 1] * 8 + [64 * long - 3] * alone, stream=3, shared=True)
    assert (batch._s is not None) == shares


def test_forks_are_runs(dev, monkeypatch):  # noqa: F811
    copies = []
    monkeypatch.setattr(kv, "_copy_in", lambda d, dst, host, st: copies.append(host.copy()))
    seqs = KVSequences(small(dev))
    a = seqs.new()
    seqs.batch([a], [150], stream=3)
    b, c = seqs.fork(a), seqs.fork(a)
    batch = seqs.batch([a, b, c], stream=3, shared=True)
    assert copies[-1][-9:].reshape(3, 3).tolist() == [[0, 0, 0], [3, 1, 1], [128] * 3] and batch._s.max_runs == 1
    assert seqs.batch([a, b, c], stream=3)._s is None


def descriptions():
    cache = kv._Cache(codes=4096, exps=4096, page_table=4096, kv_lens=4096, q_starts=4096, status=0, device=0,
                      pages=9, kv_heads=2, head_dim=64, page_size=64, seqs=4, table_width=2, tokens=4, max_q=1)
    return cache, kv._Shared(4096, 1, 4), kv._Attend(plan=4096, plan_bytes=1 << 20, heads=4)


@pytest.mark.parametrize("kw,says", [
    ({"max_runs": -1}, "max_runs"), ({"max_runs": 5}, "max_runs"), ({"max_tokens": -1}, "max_tokens"),
    ({"max_tokens": 5}, "max_tokens"), (None, "shared"),
])
def test_library_refusals(kw, says):
    from ptxgen.runtime import load_library
    L = load_library()
    cache, shared, args = descriptions()
    for k, v in (kw or {}).items():
        setattr(shared, k, v)
    ref = None if kw is None else C.byref(shared)
    ws, plan = C.c_uint64(), C.c_uint64()
    for rc in (L.emmy_kv8_attend_shared_sizes(C.byref(cache), ref, 4, C.byref(ws), C.byref(plan)),
               L.emmy_kv8_attend_shared_plan(C.byref(cache), ref, C.byref(args), None),
               L.emmy_kv8_attend_shared(C.byref(cache), ref, C.byref(args), None)):
        assert rc == -3 and says.encode() in L.emmy_last_error()
    assert L.emmy_kv8_attend_shared_sizes(None, ref, 4, C.byref(ws), C.byref(plan)) == -3
