"""The cache's host side where calls meet: collections inside its own locks,
streams whose handles say too little, graphs that outlive a call, other current
devices."""

import threading

import pytest

from ptxgen import kvcache as kv
from ptxgen.kvcache import DeviceArray, KVSequences
from ptxgen.runtime import EmmyError
from ptxgen.kvcache import DeviceArray, KVCache, KVSequences
from tests.test_kvcache import dev, small  # noqa: F401 - a fixture


def ends(work):
    """Whether ``work`` returns within some seconds."""
    t = threading.Thread(target=work, daemon=True)
    t.start()
    t.join(10)
    return not t.is_alive()


def test_a_batch_that_goes_while_buffers_are_given_or_taken(dev):  # noqa: F811
    """A collection may run anywhere, so a batch may be closed by the thread
    that holds the spare buffers' lock."""
    cache = small(dev)
    pool = kv._Pool.of(dev)

    class Held(dict):                                # as if a collection ran just there
        victims = []

        def get(self, *a):
            while self.victims:
                self.victims.pop().close()
            return super().get(*a)

        def setdefault(self, *a):
            while self.victims:
                self.victims.pop().close()
            return super().setdefault(*a)
    pool.held = Held()
    first = cache.batch([[1]], [9])
    Held.victims.append(cache.batch([[1]], [9]))
    assert ends(first.close)
    Held.victims.append(cache.batch([[1]], [9]))
    assert ends(lambda: cache.batch([[1]], [9]).close())
    assert not Held.victims and pool.bytes == sum(k[1] * len(v) for k, v in pool.held.items())


def arrays():
    return DeviceArray(1 << 20, "bf16", (1, 4, 64)), DeviceArray(1 << 21, "bf16", (1, 4, 64))


def used_and_closed(cache, stream):
    b = cache.batch([[1]], [9], stream=stream)
    b.attend(0, *arrays(), stream=stream)
    held = {p for p, _ in b._held}
    b.close()
    return held


def test_a_handle_that_comes_again_is_another_stream(dev):  # noqa: F811
    """Buffers of a stream that was destroyed, perhaps with work queued, do
    not go to the next one with its handle."""
    ids = {77: 1000}
    dev.L.emmy_stream_id = lambda st, word: setattr(word._obj, "value", ids[st]) or 0
    cache = small(dev)
    first = used_and_closed(cache, 77)
    assert used_and_closed(cache, 77) == first
    ids[77] = 1001                                   # destroyed, and made anew
    assert not used_and_closed(cache, 77) & first


def test_the_per_thread_default_stream(dev):  # noqa: F811
    """One handle, a stream in each thread: buffers stay with their thread,
    and a batch with the thread that made it."""
    dev.L.emmy_stream_id = lambda st, word: setattr(word._obj, "value", threading.get_ident() if st == 2 else 5) or 0
    cache, got = small(dev), []
    mine = used_and_closed(cache, 2)
    assert ends(lambda: got.append(used_and_closed(cache, 2))) and not got[0] & mine
    assert used_and_closed(cache, 2) == mine
    b = cache.batch([[1]], [9], stream=2)
    b.attend(0, *arrays(), stream=2)

    def elsewhere():
        with pytest.raises(EmmyError, match="per-thread"):
            b.attend(0, *arrays(), stream=2)
        got.append("refused")
    assert ends(elsewhere) and got[-1] == "refused"
    with pytest.raises(EmmyError, match="per-thread"):
        b.attend(0, *arrays(), stream=9)
    b = cache.batch([[1]], [9], stream=9)            # one of another stream waits in each thread
    dev.L.calls.clear()
    for _ in range(2):
        b.attend(0, *arrays(), stream=2)
    assert ends(lambda: b.attend(0, *arrays(), stream=2))
    assert [a[0] for name, a in dev.L.calls if name == "emmy_stream_wait_event"] == [2, 2]


def test_spare_buffers_of_streams_that_are_gone_make_room(dev, monkeypatch):  # noqa: F811
    monkeypatch.setattr(kv._Pool, "MOST", 3 * 4096)
    cache = small(dev)
    for stream in (1, 3, 4, 5, 6):
        cache.batch([[1]], [9], stream=stream).close()
    pool = kv._Pool.of(dev)
    assert {k[2] for k in pool.held} == {4, 5, 6} and pool.bytes == 3 * 4096
    assert len(dev.live - set(cache._own)) == 3


def test_buffers_that_a_graph_was_given_are_not_used_again(dev):  # noqa: F811
    """The graph may be running, on a stream that the batch never saw, when the
    batch goes: freeing waits for it, the next batch would not."""
    calls = [0]
    dev.L.emmy_kv8_captured = lambda word: setattr(word._obj, "value", calls[0]) or 0
    cache = small(dev)
    b = cache.batch([[1]], [9], stream=5)
    b.attend(0, *arrays(), stream=5)
    calls[0] += 1                                    # one more call, into a capture of stream 5
    held = {p for p, _ in b._held}
    b.close()
    assert not held & dev.live and not kv._Pool.of(dev).bytes
    first = used_and_closed(cache, 5)                # made after: as ever
    assert used_and_closed(cache, 5) == first


def test_a_collection_frees_nothing_at_once(dev):  # noqa: F811
    """It may come while some stream is captured."""
    cache = small(dev)
    b = cache.batch([[1]], [9], stream=5)
    b.attend(0, *arrays(), stream=6)
    held = {p for p, _ in b._held}
    del b
    assert held <= dev.live
    cache.batch([[1]], [9], stream=7)
    assert not held & dev.live


def test_page_moves_of_a_captured_stream_are_refused(dev):  # noqa: F811
    """A graph would make the copies at each replay, from and to pages that
    belong to others by then, while the books move on once."""
    cache = small(dev)
    seqs = KVSequences(cache)
    a = seqs.new()
    seqs.batch([a], [70])
    b, c = seqs.fork(a), seqs.new()
    seqs.batch([c], [65])
    seqs.free(a)
    d = seqs.fork(b)

    def books():
        return [seqs.pages(s) for s in (b, c, d)], [seqs.length(s) for s in (b, c, d)], list(seqs._refs), list(seqs._free)
    before = books()
    dev.L.calls.clear()
    dev.L.emmy_stream_capturing = lambda st, word: setattr(word._obj, "value", 1) or 0
    with pytest.raises(EmmyError, match="captured"):
        seqs.batch([b, d], stream=5)                 # a shared page would be copied
    assert books() == before
    seqs.free(b)
    seqs.free(d)
    before = [seqs.pages(c)], [seqs.length(c)], list(seqs._refs), list(seqs._free)
    with pytest.raises(EmmyError, match="captured"):
        seqs.compact(stream=5)                       # c's pages would move
    assert before == ([seqs.pages(c)], [seqs.length(c)], list(seqs._refs), list(seqs._free))
    assert not [name for name, _ in dev.L.calls if name == "emmy_kv8_copy_pages"]


def test_an_update_that_raises_anything_keeps_what_append_knows(dev):  # noqa: F811
    cache = small(dev)
    b = cache.batch([[1], [2]], [9, 9])
    x = DeviceArray(1 << 20, "bf16", (2, 2, 64))
    with pytest.raises(AttributeError):
        b.update([[1], [1]], [9, 9], stream="no stream")
    b.append(0, x, x)                                # the device still holds two pages


def test_the_callers_current_device_stays(dev, monkeypatch):  # noqa: F811
    """All that goes by the current device happens with the cache's as that
    one, and the caller's is back after each call."""
    now = [3]
    by_device = {"alloc", "free", "emmy_memcpy_htod", "emmy_memcpy_dtoh", "emmy_memset_d32", "event", "memset32",
                 "emmy_event_record", "emmy_stream_wait_event", "emmy_stream_sync", "emmy_stream_capturing",
                 "emmy_stream_id", "sync"}
    seen = set()

    def enter(device, word):
        word._obj.value = now[0]
        now[0] = device
        return 0

    def leave(before):
        now[0] = before
        return 0
    dev.L.emmy_device_enter, dev.L.emmy_device_leave = enter, leave

    def watched(name, call):
        def f(*a):
            assert now[0] == 1, name
            seen.add(name)
            return call(*a)
        return f
    for name in by_device:
        at = dev.L if name.startswith("emmy") else dev
        setattr(at, name, watched(name, getattr(at, name)))
    monkeypatch.setattr(kv.Device, "get", classmethod(lambda cls, ordinal=0: watched("get", lambda: dev)()))
    cache = small(dev, device=1)
    seqs = KVSequences(cache)
    a = seqs.new()
    b = seqs.batch([a], [1], stream=5)
    q, out = (DeviceArray(1 << n, "bf16", (1, 4, 64), None, 1) for n in (20, 21))
    k = DeviceArray(1 << 22, "f32", (1, 2, 64), None, 1)
    for call in (lambda: b.append(0, k, k, stream=6), lambda: b.attend(0, q, out, stream=7),
                 lambda: b.update([[1]], [2], stream=8), lambda: b.reserve(8, stream=5),
                 lambda: b.check_errors(stream=5), b.close, lambda: seqs.batch([a], stream=5),
                 lambda: seqs.compact(), cache.close):
        call()
        assert now[0] == 3
    assert seen >= by_device - {"sync"}


def test_another_stream_does_not_join_a_capture(dev):  # noqa: F811
    """A stream that waits for one that is captured becomes part of the graph."""
    cache = small(dev)
    b = cache.batch([[1]], [9], stream=5)
    b.reserve(4, stream=5)
    dev.L.emmy_stream_capturing = lambda st, word: setattr(word._obj, "value", int(st == 5)) or 0
    dev.L.calls.clear()
    with pytest.raises(EmmyError, match="captured"):
        b.attend(0, *arrays(), stream=6)
    assert not [name for name, _ in dev.L.calls if name in ("emmy_event_record", "emmy_kv8_attend")]
    b.attend(0, *arrays(), stream=5)                 # the capture goes on
    dev.L.emmy_stream_capturing = lambda st, word: setattr(word._obj, "value", int(st == 6)) or 0
    b.attend(0, *arrays(), stream=6)                 # into a capture that does not wait
    b.attend(0, *arrays(), stream=7)
    assert [a[0] for name, a in dev.L.calls if name == "emmy_stream_wait_event"] == [7]
