"""A paged 8-bit key/value cache and the attention that reads it.

The compiled attention kernels recompute nothing but keep nothing either: a
caller that generates tokens one at a time needs the keys and values of all
earlier tokens again at each step.  ``KVCache`` holds them on one GPU, one
byte a value, in pages that sequences share and exchange; its kernels are
hand-written CUDA in ``libemmyrt.so`` (``emmy_kv8_*`` in ``emmyrt.h``).  The
reference has no counterpart.

    cache = KVCache(pages=4096, kv_heads=8, head_dim=128, layers=32)
    seqs = KVSequences(cache)                 # page bookkeeping on the host
    a = seqs.new()
    batch = seqs.batch([a], [prompt_tokens])  # room for the prompt
    for layer in range(32):
        ...
        batch.append(layer, k, v)             # [tokens, kv_heads, head_dim]
        batch.attend(layer, q, out)           # [tokens, heads, head_dim]
    b = seqs.fork(a)                          # shares a's pages; copied on write
    batch = seqs.batch([a, b])                # one more token each

A held value is an e4m3 code times 2**e, with one exponent e for each page,
side (K or V) and kv head; ``append`` picks the smallest e in [-32, 63] that
holds the page's largest finite magnitude and re-rounds a page's older codes
when a new token needs a larger one.  Query i of the n new tokens of a
sequence of L keys sees key j <= L - n + i, and with a window W only those
with L - n + i - j < W or j < sinks.

Arrays are device arrays: anything with ``data_ptr()``, ``stride()``,
``get_device()``, ``shape`` and ``dtype`` as torch tensors have them, or a
``DeviceArray`` over a raw address.  No gradients are recorded.  Calls are
queued on ``stream`` (an address, or an object with ``cuda_stream``; default
the device's stream, ``Device.stream``; 0 is the legacy default stream),
return at once and allocate nothing after the first ``attend`` of a batch;
they leave the thread's current device as it was;
the caller keeps the arrays alive until the work is done and orders streams,
as with every other call here (a batch used on a stream other than the one it
was made on waits for that once).
"""

from __future__ import annotations

import ctypes as C
import functools
import threading
import weakref
from array import array

import numpy as np

from .runtime import Device, EmmyError, check, load_library

E_MIN, E_MAX = -32, 63
HEAD_DIMS = (64, 128)
PAGE_SIZES = (64, 128, 256)
MAX_SEQS = 4096
MAX_PAIRS = 480            # pages a launch of copy_pages takes
WORKSPACE_ZERO = 16384     # bytes of a workspace that start as zeros
PER_THREAD = 2             # the per-thread default stream's handle

STATUS = {0x401: "a page number outside the pool",
          0x402: "a sequence longer than its row of the table, or more new tokens than keys or rows",
          0x403: "a bounded wait inside a kernel ran out",
          0x404: "a plan that was made for another call"}


class _Cache(C.Structure):
    """``emmy_kv8``."""
    _fields_ = [(n, C.c_uint64) for n in ("codes", "exps", "page_table", "kv_lens", "q_starts",
                                          "status")] \
        + [(n, C.c_int32) for n in ("device", "pages", "kv_heads", "head_dim", "page_size",
                                    "seqs", "table_width", "tokens", "max_q")]


class _Attend(C.Structure):
    """``emmy_kv8_attend_args``."""
    _fields_ = [("q", C.c_uint64), ("out", C.c_uint64), ("workspace", C.c_uint64),
                ("plan", C.c_uint64), ("workspace_bytes", C.c_uint64), ("plan_bytes", C.c_uint64),
                ("q_strides", C.c_int64 * 2),
                ("out_strides", C.c_int64 * 2), ("dtype", C.c_int32), ("heads", C.c_int32),
                ("window", C.c_int32), ("sinks", C.c_int32), ("scale", C.c_float)]


_Strides = C.c_int64 * 2


class DeviceArray:
    """A view of device memory at a raw address: ``dtype`` one of "f32",
    "bf16", "f16", "u8", "i8"; strides in elements, row-major by default."""

    def __init__(self, ptr: int, dtype: str, shape, strides=None, device: int = 0):
        self.ptr, self.dtype, self.shape, self.device = int(ptr), dtype, tuple(shape), device
        if strides is None:
            strides, n = [], 1
            for s in reversed(self.shape):
                strides.append(n)
                n *= s
            strides.reverse()
        self.strides = tuple(strides)

    def data_ptr(self) -> int:
        return self.ptr

    def stride(self) -> tuple:
        return self.strides

    def get_device(self) -> int:
        return self.device


_DTYPES = {"f32": 0, "bf16": 1, "f16": 2, "u8": 3, "i8": 4}
_NAMES = {"float32": "f32", "bfloat16": "bf16", "float16": "f16", "half": "f16", "uint8": "u8",
          "int8": "i8", "float8_e4m3fn": "u8"}


def _dtype_code(dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        name = str(dtype).split(".")[-1]
        code = _DTYPES.get(_NAMES.get(name, name))
        if code is None:
            raise EmmyError(f"unsupported dtype {dtype}")
        _DTYPES[dtype] = code
    return code


def _stream_of(stream, dev: Device) -> int:
    if type(stream) is int:
        return stream
    if stream is None:
        stream = dev.stream
    stream = getattr(stream, "cuda_stream", stream)
    return stream if isinstance(stream, int) else stream.value or 0


class _Current:
    """A device as the thread's current one for a scope: what allocates, copies
    and records here goes by that, and callers find their own back."""

    def __init__(self, L, ordinal: int):
        self.L, self.ordinal = L, ordinal

    def __enter__(self):
        word = C.c_int()
        check(self.L.emmy_device_enter(self.ordinal, C.byref(word)), "device")
        self.before = word.value

    def __exit__(self, *exc):
        if self.before != self.ordinal:
            self.L.emmy_device_leave(self.before)


def _at_home(method):
    """A method of a cache or batch, with its device the current one."""
    @functools.wraps(method)
    def call(self, *a, **kw):
        with _Current(self.L, self.ordinal):
            return method(self, *a, **kw)
    return call


def _stream_id(dev: Device, st: int) -> int:
    """Of the stream itself: handles of destroyed streams come again, and
    PER_THREAD is another stream in each thread."""
    word = C.c_uint64()
    check(dev.L.emmy_stream_id(st, C.byref(word)), "stream")
    return word.value or st


def _capturing(dev: Device, st: int) -> bool:
    word = C.c_int()
    check(dev.L.emmy_stream_capturing(st, C.byref(word)), "stream")
    return word.value != 0


def _captured(dev: Device) -> int:
    """Calls of this process that went into captures so far."""
    word = C.c_uint64()
    check(dev.L.emmy_kv8_captured(C.byref(word)), "captured calls")
    return word.value


def _outside_capture(dev: Device, st: int, why: str) -> None:
    """A graph would keep the address of host memory that is gone when it
    runs, or do what later calls count on only then."""
    if _capturing(dev, st):
        raise EmmyError(f"not while the stream is captured: {why}")


# Device's own copy calls take a null stream for "the device's"; these take the
# handle as it is, 0 included.
def _copy_in(dev: Device, dst: int, host: np.ndarray, st: int) -> None:
    check(dev.L.emmy_memcpy_htod(dst, host.ctypes.data, host.nbytes, st), "htod")


def _ints(x, name: str) -> np.ndarray:
    a = np.asarray(x)
    if a.size == 0:
        return a.astype(np.int64)
    if a.dtype.kind not in "iu":
        raise EmmyError(f"{name} must be whole numbers")
    return a.astype(np.int64)


class _Pool:
    """Buffers of closed batches on one device, by (use, bytes, the id of the
    one stream they were used on): the next batch on that stream takes them
    with no wait.  Kept for the process, up to ``MOST`` bytes; those of the
    stream that was first kept go first."""

    MOST = 512 << 20

    @classmethod
    def of(cls, dev: Device, ordinal: int = 0) -> "_Pool":
        return dev.__dict__.get("_kv_pool") or dev.__dict__.setdefault("_kv_pool", cls(dev, ordinal))

    def __init__(self, dev: Device, ordinal: int):
        self.dev, self.ordinal, self.held, self.bytes, self.gone = dev, ordinal, {}, 0, []
        self.lock = threading.RLock()   # a collection inside of it may close a batch

    def take(self, use: str, nbytes: int, stream: int, sid: int) -> tuple[int, tuple]:
        """(address, key to give it back by) of a buffer for work on ``stream``,
        whose id is ``sid``."""
        key = (use, 1 << max(12, (nbytes - 1).bit_length()), sid)
        if self.gone:
            self.drain()
        with self.lock:
            held = self.held.get(key)
            if held:
                self.bytes -= key[1]
                return held.pop(), key
        ptr = self.dev.alloc(key[1])
        if use == "workspace":
            check(self.dev.L.emmy_memset_d32(ptr, 0, WORKSPACE_ZERO // 4, stream), "memset")
        return ptr, key

    def drain(self) -> None:
        """Free what is not to be used again: waits for what still runs on it."""
        with _Current(self.dev.L, self.ordinal):
            while self.gone:
                try:
                    ptr = self.gone.pop()
                except IndexError:      # another thread's turn
                    break
                self.dev.free(ptr)

    def give(self, ptr: int, key: tuple, reuse: bool, later: bool = False) -> None:
        """``later``: what is to be freed is at the next call of ``take``, for a
        collection may come while some stream is captured, and memory that is
        freed then ends the capture."""
        with self.lock:
            if reuse and self.bytes + key[1] > self.MOST:
                self._make_room(key)
            if reuse and self.bytes + key[1] <= self.MOST:
                self.held.setdefault(key, []).append(ptr)
                self.bytes += key[1]
            else:
                self.gone.append(ptr)
        if self.gone and not later:
            self.drain()

    def _make_room(self, key: tuple) -> None:
        for other in [k for k in self.held if k[2] != key[2]]:
            spare = self.held.get(other)
            while spare and self.bytes + key[1] > self.MOST:
                self.gone.append(spare.pop())
                self.bytes -= other[1]
            if not spare:
                self.held.pop(other, None)


class KVCache:
    """``layers`` layers of ``pages`` pages of ``page_size`` tokens each, on
    one GPU.  ``storage``: (codes, exps) to adopt instead of allocating --
    contiguous 8-bit arrays [layers, pages, 2, kv_heads, page_size, head_dim]
    (e4m3 codes; K, then V) and [layers, pages, 2, kv_heads] (int8)."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 layers: int = 1, device: int = 0, storage=None):
        if head_dim not in HEAD_DIMS:
            raise EmmyError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if page_size not in PAGE_SIZES:
            raise EmmyError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if not 1 <= kv_heads <= 1024:
            raise EmmyError(f"kv_heads must be between 1 and 1024, got {kv_heads}")
        if not 1 <= pages < 2 ** 31:
            raise EmmyError(f"pages must be between 1 and 2^31 - 1, got {pages}")
        if not 1 <= layers <= 65535:
            raise EmmyError(f"layers must be between 1 and 65535, got {layers}")
        self.pages, self.kv_heads, self.head_dim = pages, kv_heads, head_dim
        self.page_size, self.layers, self.ordinal = page_size, layers, device
        self.layer_codes = pages * 2 * kv_heads * page_size * head_dim
        self.layer_exps = pages * 2 * kv_heads
        self._own: list[int] = []
        self._storage = storage
        if storage is not None:
            codes, exps = storage
            shape = (layers, pages, 2, kv_heads, page_size, head_dim)
            for name, x, want, types in (("codes", codes, shape, (3, 4)),
                                         ("exps", exps, shape[:4], (4,))):
                if tuple(x.shape) != want:
                    raise EmmyError(f"storage: {name} has shape {tuple(x.shape)}, expected {want}")
                if _dtype_code(x.dtype) not in types:
                    raise EmmyError(f"storage: {name} must be an 8-bit array, got {x.dtype}")
                n = 1
                for size, stride in zip(reversed(want), reversed(tuple(x.stride()))):
                    if size != 1 and stride != n:
                        raise EmmyError(f"storage: {name} must be contiguous")
                    n *= size
                if x.get_device() != device:
                    raise EmmyError(f"storage: {name} is not on device {device}")
            self.codes, self.exps = codes.data_ptr(), exps.data_ptr()
            if self.codes % 16:
                raise EmmyError("storage: codes must be 16-byte aligned")
        self.L = load_library()
        with _Current(self.L, device):
            self._open(storage is None)
        self._cdesc = self._desc()
        self._cref = C.byref(self._cdesc)

    def _open(self, allocate: bool) -> None:
        layers = self.layers
        self.dev = Device.get(self.ordinal)
        if allocate:
            _Pool.of(self.dev, self.ordinal).drain()
            for attr, n in (("codes", layers * self.layer_codes), ("exps", layers * self.layer_exps)):
                ptr = self.dev.alloc(n)
                self._own.append(ptr)
                setattr(self, attr, ptr)
            # pages that nothing wrote hold zeros
            self.dev.memset32(self.codes, 0, (layers * self.layer_codes + 3) // 4)
            self.dev.memset32(self.exps, 0, (layers * self.layer_exps + 3) // 4)
            self.dev.sync()

    def _desc(self) -> _Cache:
        d = _Cache()
        d.codes, d.exps, d.device = self.codes, self.exps, self.ordinal
        d.pages, d.kv_heads = self.pages, self.kv_heads
        d.head_dim, d.page_size = self.head_dim, self.page_size
        return d

    def batch(self, page_table, kv_lens, q_lens=None, stream=None) -> "Batch":
        """The sequences of one step: ``page_table`` [seqs, width] page
        numbers, ``kv_lens`` keys of each sequence with its new tokens,
        ``q_lens`` new tokens of each (default 1).  Host arrays, checked
        here and copied to the device on ``stream``."""
        return Batch(self, page_table, kv_lens, q_lens, stream)

    def copy_pages(self, src, dst, stream=None) -> None:
        """Copy pages ``src[i]`` to ``dst[i]`` in every layer (host lists);
        no page twice in ``dst`` nor in both lists."""
        try:
            src, dst = array("i", src), array("i", dst)
        except (TypeError, OverflowError) as exc:
            raise EmmyError(f"copy_pages: src and dst are lists of page numbers: {exc}") from None
        n = len(src)
        if n != len(dst):
            raise EmmyError("copy_pages: src and dst are lists of the same length")
        if n == 0:
            return
        if min(src) < 0 or min(dst) < 0 or max(src) >= self.pages or max(dst) >= self.pages:
            raise EmmyError(f"copy_pages: a page is outside 0..{self.pages - 1}")
        targets = set(dst)
        if len(targets) != n:
            raise EmmyError("copy_pages: a page is in dst twice")
        if not targets.isdisjoint(src):
            raise EmmyError("copy_pages: a page is in both src and dst")
        if not self.codes:
            raise EmmyError("the cache is closed")
        st = _stream_of(stream, self.dev)
        at, to = src.buffer_info()[0], dst.buffer_info()[0]
        for i in range(0, n, MAX_PAIRS):
            rc = self.L.emmy_kv8_copy_pages(self._cref, self.layers, at + 4 * i, to + 4 * i,
                                            min(MAX_PAIRS, n - i), st)
            if rc:
                check(rc, "copy_pages")

    @_at_home
    def close(self) -> None:
        """Free what this cache allocated (not adopted storage)."""
        own, self._own = self._own, []
        self.codes = self.exps = 0
        for p in own:
            self.dev.free(p)

    def __del__(self):
        try:
            self.close()
        except Exception:  # the context may be gone when the process ends
            pass


class Batch:
    """One step's sequences on the device.  Rows of the arrays given to
    ``append`` and ``attend`` are the new tokens, sequence after sequence;
    rows behind the last one are left alone.  Calls of one batch share a
    workspace, so they must not overlap on the GPU: two captured graphs, or
    two streams, that run at once need a batch each.  One made on the
    per-thread default stream is for that thread and stream.  A graph captured over
    ``append`` and ``attend`` replays with what ``update`` last put there; the
    batch has to live as long as the graph may run.  Making, ``reserve`` (or
    the first ``attend`` with some heads, window and sinks), ``update`` and
    ``check_errors`` stay outside of captures."""

    def __init__(self, cache: KVCache, page_table, kv_lens, q_lens=None, stream=None):
        self.cache, self.dev, self.L, self.ordinal = cache, cache.dev, cache.L, cache.ordinal
        self._make(page_table, kv_lens, q_lens, stream)

    @_at_home
    def _make(self, page_table, kv_lens, q_lens, stream) -> None:
        cache = self.cache
        table = _ints(page_table, "page_table")
        if table.ndim != 2 or table.shape[0] < 1 or table.shape[1] < 1:
            raise EmmyError("page_table must be [sequences, pages]")
        if table.shape[0] > MAX_SEQS:
            raise EmmyError(f"a batch holds at most {MAX_SEQS} sequences")
        self.seqs, self.width = table.shape
        if self.width * cache.page_size > 2 ** 30:
            raise EmmyError("a sequence holds at most 2^30 keys")
        self.tokens = self.max_q = None
        self._buf = 0
        self._held: list[tuple[int, tuple]] = []   # buffers of this batch, to give back
        self._ws: tuple[int, int] = (0, 0)         # workspace: address, bytes
        self._plans: dict[tuple, tuple] = {}       # (heads, window, sinks): plan address and bytes
        self._stale = False
        host = self._packed(table, kv_lens, q_lens)
        self._stream, self._reuse = _stream_of(stream, self.dev), True
        _outside_capture(self.dev, self._stream, "lengths and page numbers are copied from the host")
        self._pool, self._captured = _Pool.of(self.dev, cache.ordinal), _captured(self.dev)
        self._id = _stream_id(self.dev, self._stream)
        self._who = self._id if self._stream == PER_THREAD else self._stream
        self._others: set[int] = set()             # further streams it was used on
        self._buf = self._take("batch", host.nbytes, self._stream)
        _copy_in(self.dev, self._buf, host, self._stream)
        d = self._d = cache._desc()
        d.status = self._buf
        d.kv_lens = self._buf + 16
        d.q_starts = d.kv_lens + 4 * self.seqs
        d.page_table = d.q_starts + 4 * (self.seqs + 1)
        d.seqs, d.table_width, d.tokens, d.max_q = self.seqs, self.width, self.tokens, self.max_q
        self._ref, self._layer = C.byref(d), 0
        self._a = _Attend()
        self._aref = C.byref(self._a)
        self._ks, self._vs = _Strides(), _Strides()
        self._append, self._attend = self.L.emmy_kv8_append, self.L.emmy_kv8_attend

    def _take(self, use: str, nbytes: int, st: int) -> int:
        held = self._pool.take(use, nbytes, st, self._id if st == self._stream else _stream_id(self.dev, st))
        self._held.append(held)
        return held[0]

    def _on(self, stream) -> int:
        """The handle of ``stream``; one other than the batch's own waits, the
        first time, for what is queued on that (its lengths, a page copy).
        One that is being captured cannot wait: its graph is replayed after."""
        st = _stream_of(stream, self.dev)
        who = st if st != PER_THREAD else _stream_id(self.dev, st)
        if who != self._who and who not in self._others:
            if self._stream == PER_THREAD:
                raise EmmyError("a batch made on the per-thread default stream is for that thread and stream")
            self._reuse = False
            with _Current(self.L, self.ordinal):
                if _capturing(self.dev, st):
                    return st
                _outside_capture(self.dev, self._stream,
                                 "another stream that waited for it would become part of the graph")
                ev = self.dev.event()
                try:
                    check(self.L.emmy_event_record(ev, self._stream), "event record")
                    check(self.L.emmy_stream_wait_event(st, ev), "stream wait event")
                finally:
                    self.L.emmy_event_destroy(ev)
            self._others.add(who)
        return st

    def _packed(self, table, kv_lens, q_lens) -> np.ndarray:
        """Checked lengths and table as one int32 array: status word and
        padding, kv_lens, q_starts, table."""
        P, B = self.cache.page_size, self.seqs
        kv = _ints(kv_lens, "kv_lens").reshape(-1)
        q = np.ones(B, np.int64) if q_lens is None else _ints(q_lens, "q_lens").reshape(-1)
        if len(kv) != B or len(q) != B or table.shape != (B, self.width):
            raise EmmyError(f"expected {B} lengths and a page table [{B}, {self.width}]")
        if (q < 0).any() or (q > kv).any():
            raise EmmyError("a sequence has between 0 and its kv_len new tokens")
        if (kv > self.width * P).any():
            raise EmmyError(f"a sequence is longer than its {self.width} pages of {P} tokens")
        used = np.arange(self.width) < -(-kv // P)[:, None]
        if ((table < 0) | (table >= self.cache.pages))[used].any():
            raise EmmyError(f"page_table: a page is outside 0..{self.cache.pages - 1}")
        tokens, most = int(q.sum()), int(q.max())
        if tokens >= 2 ** 31:
            raise EmmyError("too many new tokens")
        if self.tokens is None:
            self.tokens, self.max_q = tokens, most
        elif tokens > self.tokens or most > self.max_q:
            raise EmmyError(f"update: the batch was made for {self.tokens} new tokens, "
                            f"at most {self.max_q} of a sequence")
        # pages that append writes: of no more than one sequence
        span = np.arange(self.width)
        written = table[(span >= ((kv - q) // P)[:, None]) & (span <= ((kv - 1) // P)[:, None])
                        & (q > 0)[:, None]]
        # (np.unique costs 6 us however few there are)
        self._clash = len(set(written.tolist()) if len(written) < 256 else np.unique(written)) != len(written)
        host = np.zeros(4 + 2 * B + 1 + B * self.width, np.int32)
        host[4:4 + B] = kv
        host[5 + B:5 + 2 * B] = np.cumsum(q)
        host[5 + 2 * B:] = np.where(used, table, 0).reshape(-1)
        return host

    @_at_home
    def update(self, page_table, kv_lens, q_lens=None, stream=None) -> None:
        """New contents in the same device arrays, for the next replay of a
        graph or the next step: as many sequences, a table as wide, no more
        new tokens than the batch was made for."""
        self._live()
        clash = self._clash
        try:
            host = self._packed(_ints(page_table, "page_table"), kv_lens, q_lens)
            st = self._on(stream)
            _outside_capture(self.dev, st, "lengths and page numbers are copied from the host")
            _copy_in(self.dev, self._buf + 16, host[4:], st)
        except BaseException:
            self._clash = clash         # of what the device still holds
            raise
        for key in self._plans:
            self._plan(key, st)
        self._stale = False

    def _live(self) -> None:
        if not self._buf:
            raise EmmyError("the batch is closed")

    def _usable(self, layer: int) -> None:
        self._live()
        if self._stale:
            raise EmmyError("the batch names pages that compact() moved: update it or make a new one")
        if not 0 <= layer < self.cache.layers:
            raise EmmyError(f"layer {layer} is outside 0..{self.cache.layers - 1}")
        c = self.cache
        if not c.codes:
            raise EmmyError("the cache is closed")
        if layer != self._layer:
            d = self._d
            d.codes = c.codes + layer * c.layer_codes
            d.exps = c.exps + layer * c.layer_exps
            self._layer = layer

    def _array(self, x, name: str, heads: int | None):
        """(address, dtype code, (token, head) strides, heads) of a
        [tokens, heads, head_dim] argument."""
        shape, stride = x.shape, x.stride()
        if len(shape) != 3 or shape[0] < self.tokens or shape[2] != self.cache.head_dim \
                or (heads is not None and shape[1] != heads):
            raise EmmyError(f"{name} has shape {tuple(shape)}, expected "
                            f"[>= {self.tokens}, {heads or 'heads'}, {self.cache.head_dim}]")
        if stride[2] != 1:
            raise EmmyError(f"{name}: the last dimension must be contiguous")
        if x.get_device() != self.cache.ordinal:
            raise EmmyError(f"{name} is not on device {self.cache.ordinal}")
        code = _DTYPES.get(x.dtype)
        return x.data_ptr(), _dtype_code(x.dtype) if code is None else code, stride, shape[1]

    def append(self, layer: int, k, v, stream=None) -> None:
        """Write the new tokens' keys and values (f32, bf16 or f16) into
        their pages of ``layer``."""
        self._usable(layer)
        if self._clash:
            raise EmmyError("append: two sequences of the batch write to the same page")
        kp, kt, ks, _ = self._array(k, "k", self.cache.kv_heads)
        vp, vt, vs, _ = self._array(v, "v", self.cache.kv_heads)
        if kt != vt or kt > 2:
            raise EmmyError("append: k and v must both be f32, bf16 or f16")
        sk, sv = self._ks, self._vs
        sk[0], sk[1], sv[0], sv[1] = ks[0], ks[1], vs[0], vs[1]
        rc = self._append(self._ref, kp, vp, kt, sk, sv, self._on(stream))
        if rc:
            check(rc, "append")

    def reserve(self, heads: int, window: int = 0, sinks: int = 0, stream=None) -> None:
        """What ``attend`` needs for ``heads`` query heads, a window and sinks
        besides its arrays: workspace and plan.  The first call does it
        otherwise; before a graph is captured it has to be done."""
        self._live()
        key = (heads, window, sinks)
        if key not in self._plans:
            self._reserve(key, stream)

    @_at_home
    def _reserve(self, key: tuple, stream) -> None:
        heads, window, sinks = key
        if not 0 <= window < 2 ** 31 or not 0 <= sinks < 2 ** 31:
            raise EmmyError("attend: window and sinks are between 0 and 2^31 - 1")
        if not 1 <= heads <= 2 ** 20:
            raise EmmyError(f"attend: {heads} query heads")
        st = self._on(stream)
        _outside_capture(self.dev, st, "reserve() for these heads, window and sinks comes before")
        ws, plan = C.c_uint64(), C.c_uint64()
        check(self.L.emmy_kv8_attend_sizes(self._ref, heads, C.byref(ws), C.byref(plan)), "attend")
        if ws.value > self._ws[1]:
            self._ws = self._take("workspace", ws.value, st), ws.value
        self._plans[key] = self._take("plan", plan.value, st), plan.value
        try:
            self._plan(key, st)
        except EmmyError:
            del self._plans[key]
            raise

    def _plan(self, key: tuple, st: int) -> None:
        a = self._a
        a.heads, a.window, a.sinks = key
        a.plan, a.plan_bytes = self._plans[key]
        check(self.L.emmy_kv8_attend_plan(self._ref, self._aref, st), "attend")

    def attend(self, layer: int, q, out, scale: float | None = None, window: int = 0,
               sinks: int = 0, stream=None):
        """Attention of the new tokens' queries ``q`` [tokens, heads,
        head_dim] (bf16 or f16) over ``layer`` into ``out`` (same type and
        shape, not overlapping ``q``); returns ``out``.  ``scale`` defaults
        to head_dim ** -0.5.  ``window``: only the last ``window`` positions,
        and the first ``sinks`` ones (0: all)."""
        self._usable(layer)
        a = self._a
        qp, qt, qs, heads = self._array(q, "q", None)
        op, ot, os_, _ = self._array(out, "out", heads)
        if qt != ot or qt not in (1, 2):
            raise EmmyError("attend: q and out must both be bf16 or f16")
        plan = self._plans.get((heads, window, sinks))
        if plan is None:
            self.reserve(heads, window, sinks, stream)
            plan = self._plans[heads, window, sinks]
        a.q, a.out = qp, op
        a.workspace, a.workspace_bytes = self._ws
        a.plan, a.plan_bytes = plan
        a.q_strides[0], a.q_strides[1] = qs[0], qs[1]
        a.out_strides[0], a.out_strides[1] = os_[0], os_[1]
        a.dtype, a.heads, a.window, a.sinks = qt, heads, window, sinks
        a.scale = self.cache.head_dim ** -0.5 if scale is None else scale
        rc = self._attend(self._ref, self._aref, self._on(stream))
        if rc:
            check(rc, "attend")
        return out

    @_at_home
    def check_errors(self, stream=None) -> None:
        """Wait for ``stream`` and raise if a kernel of this batch reported
        something in its status word; clears it."""
        self._live()
        word = np.zeros(1, np.uint32)
        st = self._on(stream)
        _outside_capture(self.dev, st, "the status word is read on the host")
        check(self.L.emmy_memcpy_dtoh(word.ctypes.data, self._buf, 4, st), "dtoh")
        check(self.L.emmy_stream_sync(st), "stream sync")
        if word[0]:
            self._reuse = False         # its counters may not be as they should
            check(self.L.emmy_memset_d32(self._buf, 0, 1, st), "memset")
            raise EmmyError(f"cache kernel reported error 0x{word[0]:x}: "
                            f"{STATUS.get(int(word[0]), 'unknown')}")

    def close(self) -> None:
        """Give the batch's buffers back for later batches: nothing that is
        not queued yet may use them after this.  Where a graph may still be
        running that was captured while the batch lived -- on any stream -- or
        another stream was used, they are freed instead, which waits."""
        self._close(later=False)

    def _close(self, later: bool) -> None:
        held, self._held = self._held, []
        self._buf, self._ws, self._plans = 0, (0, 0), {}
        if held:
            reuse = self._reuse and _captured(self.dev) == self._captured
            for ptr, key in held:
                self._pool.give(ptr, key, reuse, later)

    def __del__(self):
        try:
            self._close(later=True)
        except Exception:  # the context may be gone when the process ends
            pass


class KVSequences:
    """Which pages of a cache hold which sequence: reference counts, copy on
    write, and the page moves of ``compact``.  Host bookkeeping; the copies
    it needs are queued on the stream given, which must be the one that
    appends, or one ordered with it."""

    def __init__(self, cache: KVCache):
        self.cache = cache
        self._refs = [0] * cache.pages
        self._free = list(range(cache.pages - 1, -1, -1))   # the lowest page is taken first
        self._pages: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0
        self._batches: list = []

    # -- sequences ----------------------------------------------------------

    def new(self) -> int:
        """An empty sequence."""
        sid, self._next = self._next, self._next + 1
        self._pages[sid], self._len[sid] = [], 0
        return sid

    def _known(self, sid: int) -> None:
        if sid not in self._pages:
            raise EmmyError(f"no sequence {sid}")

    def length(self, sid: int) -> int:
        self._known(sid)
        return self._len[sid]

    def pages(self, sid: int) -> list[int]:
        self._known(sid)
        return list(self._pages[sid])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def fork(self, sid: int) -> int:
        """A sequence with the same tokens, on the same pages; a shared page
        is copied when one of its sequences writes to it."""
        self._known(sid)
        new = self.new()
        self._pages[new], self._len[new] = list(self._pages[sid]), self._len[sid]
        for p in self._pages[new]:
            self._refs[p] += 1
        return new

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            self._free.append(page)

    def truncate(self, sid: int, length: int) -> None:
        """Forget the tokens from position ``length`` on (rejected drafts).  The
        last page keeps the scale that forgotten ones asked for, and its older
        tokens the rounding to that."""
        self._known(sid)
        if not 0 <= length <= self._len[sid]:
            raise EmmyError(f"truncate: sequence {sid} has {self._len[sid]} tokens")
        keep = -(-length // self.cache.page_size)
        for p in self._pages[sid][keep:]:
            self._drop(p)
        del self._pages[sid][keep:]
        self._len[sid] = length

    def free(self, sid: int) -> None:
        """Forget a sequence; pages no other sequence shares are free again."""
        self.truncate(sid, 0)
        del self._pages[sid], self._len[sid]

    # -- steps --------------------------------------------------------------

    def batch(self, sids, q_lens=None, stream=None) -> Batch:
        """Room for ``q_lens[i]`` (default 1) more tokens of each sequence:
        pages are taken, shared ones about to be written to copied, and the
        lengths moved on.  Where it raises (pages ran out), nothing has
        changed."""
        sids = list(sids)
        q = [1] * len(sids) if q_lens is None else [int(n) for n in _ints(q_lens, "q_lens")]
        if not sids or len(q) != len(sids):
            raise EmmyError("batch: at least one sequence, and a q_len for each")
        if len(set(sids)) != len(sids):
            raise EmmyError("batch: a sequence is named twice")
        for sid, n in zip(sids, q):
            self._known(sid)
            if n < 0:
                raise EmmyError("batch: a q_len is negative")
        P = self.cache.page_size
        refs, need, copies = {}, 0, []
        for sid, n in zip(sids, q):
            have, length = self._pages[sid], self._len[sid]
            need += max(0, -(-(length + n) // P) - len(have))
            if n and length % P:
                last = have[-1]
                held = refs.get(last, self._refs[last])
                if held > 1:
                    refs[last] = held - 1
                    copies.append(sid)
                    need += 1
        if need > len(self._free):
            raise EmmyError(f"batch: {need} pages needed, {len(self._free)} free")
        taken = self._free[:-need - 1:-1]          # the next ones, from the end
        pages = {sid: list(self._pages[sid]) for sid in sids}
        src, at = [pages[sid][-1] for sid in copies], len(copies)
        for sid, page in zip(copies, taken):
            pages[sid][-1] = page
        for sid, n in zip(sids, q):
            more = -(-(self._len[sid] + n) // P) - len(pages[sid])
            if more > 0:
                pages[sid] += taken[at:at + more]
                at += more
        lens = [self._len[sid] + n for sid, n in zip(sids, q)]
        self._outside_capture(stream)
        self.cache.copy_pages(src, taken[:len(src)], stream)
        b = Batch(self.cache, self._table(list(pages.values())), lens, q, stream)
        # the books follow once nothing can fail
        del self._free[len(self._free) - need:]
        for page in src:
            self._refs[page] -= 1
        for page in taken:
            self._refs[page] = 1
        self._pages.update(pages)
        self._len.update(zip(sids, lens))
        self._track(b)
        return b

    def _outside_capture(self, stream) -> None:
        dev = self.cache.dev
        with _Current(self.cache.L, self.cache.ordinal):
            _outside_capture(dev, _stream_of(stream, dev),
                             "the books move on once, a graph's page copies at each replay")

    def table(self, sids) -> np.ndarray:
        """Page numbers [sequences, pages of the longest], rows filled up with 0."""
        sids = list(sids)
        for sid in sids:
            self._known(sid)
        return self._table([self._pages[s] for s in sids])

    @staticmethod
    def _table(rows) -> np.ndarray:
        out = np.zeros((len(rows), max(1, max(map(len, rows), default=1))), np.int32)
        for i, r in enumerate(rows):
            out[i, :len(r)] = r
        return out

    def _track(self, batch: Batch) -> None:
        self._batches = [r for r in self._batches if r() is not None]
        self._batches.append(weakref.ref(batch))

    def compact(self, stream=None) -> int:
        """Move pages so that those in use are the first ones of the pool;
        returns how many are in use.  Batches that ``batch`` made before name
        old pages and refuse to run until updated; graphs captured over them,
        and batches of tables kept elsewhere, must not run until then."""
        used = [p for p, n in enumerate(self._refs) if n]
        n = len(used)
        holes = [p for p in range(n) if not self._refs[p]]
        moved = dict(zip([p for p in used if p >= n], holes))
        if moved:
            self._outside_capture(stream)
            self.cache.copy_pages(list(moved), list(moved.values()), stream)
            for old, new in moved.items():
                self._refs[new], self._refs[old] = self._refs[old], 0
            for pages in self._pages.values():
                pages[:] = [moved.get(p, p) for p in pages]
            for r in self._batches:
                if r() is not None:
                    r()._stale = True
        self._free = list(range(self.cache.pages - 1, n - 1, -1))
        return n
