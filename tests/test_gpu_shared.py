"""Attention over shared prefixes on the GPU against the 64-bit oracle, within the
bound of attention that shares nothing: the two softmaxes join in f32, by steps
that the bound's sums count already."""

import numpy as np
import pytest

from tests import kv8_oracle as ref
from tests.test_gpu_kvcache import NP, cache_of, gpu  # noqa: F401 - gpu is a fixture

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def share_all(monkeypatch):
    """Sharing however little it saves."""
    from ptxgen import kvcache
    monkeypatch.setattr(kvcache, "MIN_SAVED", {64: 0, 128: 0})


def layout(rng, runs, P, spare=2):
    """(table, keys, new tokens, pages) of runs [(shared keys, [(own keys, new
    tokens), ..]), ..]."""
    rows, kv, ql, at = [], [], [], 0
    for prefix, members in runs:
        first = list(range(at, at + prefix // P))
        at += prefix // P
        for own, n in members:
            more = -(-own // P)
            rows.append(first + list(range(at, at + more)))
            at += more
            kv.append(prefix + own)
            ql.append(n)
    order = rng.permutation(at + spare)
    table = np.zeros((len(rows), max(1, max(map(len, rows)))), np.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = order[r]
    return table, kv, ql, at + spare


def attend(gpu, codes, exps, table, kv, ql, q, dtype, shared=True, pad=2, runs=None, **kw):  # noqa: F811
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    batch = cache.batch(table, kv, ql, shared=shared)
    if runs is not None:
        assert (batch._s.max_runs if batch._s else 0) == runs
    rows, heads, d = q.shape
    full = np.concatenate([q, np.ones((pad, heads, d), q.dtype)])
    fill = np.full(full.shape, 77.0).astype(NP[dtype])
    got = []
    for _ in range(2):
        out = gpu.put(fill, dtype)
        batch.attend(0, gpu.put(full, dtype), out, **kw)
        got.append(gpu.get(out, fill.shape, NP[dtype]))
    batch.check_errors()
    assert got[0].tobytes() == got[1].tobytes()          # no order of arrival in it
    assert (got[0][rows:].astype(np.float32) == 77).all()
    batch.close()
    return got[0][:rows]


CASES = [
    # kv heads, group, head_dim, page, dtype, runs
    (2, 4, 128, 64, "bf16", [(64, [(1, 1), (1, 1)])]),
    (2, 4, 128, 64, "bf16", [(320, [(30, 1), (64, 1), (65, 1), (1, 1)])]),                     # row kernel first
    (1, 8, 64, 64, "f16", [(1000 // 64 * 64, [(100, 1), (3, 1)])]),
    (1, 1, 64, 128, "bf16", [(256, [(9, 2), (5, 3)])]),
    (3, 5, 128, 64, "f16", [(192, [(10, 3), (200, 3)])]),                                      # 30 rows, two blocks
    (1, 16, 64, 64, "bf16", [(128, [(70, 2), (2, 2)])]),                                       # 64 rows: tile kernel
    (2, 4, 128, 64, "bf16", [(2048, [(1 + 37 * i, 1) for i in range(20)])]),
    (1, 4, 64, 64, "f16", [(640, [(1 + i, 1) for i in range(64)])]),                           # exactly a unit
    (1, 4, 64, 64, "bf16", [(640, [(1 + i, 1) for i in range(65)])]),                          # and a row block more
    (1, 5, 128, 128, "bf16", [(1280, [(4 + 11 * i, 4) for i in range(20)])]),                  # rows across units
    (2, 7, 64, 64, "f16", [(512, [(4 + 50 * i, 1 + i % 4) for i in range(30)])]),
    (1, 32, 128, 64, "f16", [(448, [(1 + i, 1) for i in range(9)])]),
    (8, 4, 128, 64, "bf16", [(8192, [(100, 1), (7, 1), (300, 1)])]),                           # many parts
    (1, 4, 128, 256, "bf16", [(16384, [(700, 1)] * 12)]),
    # several runs, sequences by themselves, and some that sit the step out
    (2, 2, 64, 64, "bf16", [(128, [(5, 1), (70, 1)]), (0, [(33, 1)]), (256, [(1, 1)] * 30), (0, [(300, 2), (64, 0)])]),
    (1, 4, 128, 64, "f16", [(0, [(500, 1)]), (192, [(64, 0), (5, 1), (64, 0), (9, 3)]), (64, [(1, 1), (2, 1)])]),
    (1, 3, 64, 128, "f16", [(128 * n, [(1 + n, 1)] * (n + 1)) for n in range(1, 9)]),
    (4, 8, 64, 64, "bf16", [(64 * 9, [(1 + 64 * (i % 3), 4) for i in range(16)]), (64, [(200, 4)] * 3)]),
]


def name(c):
    return f"h{c[0]}x{c[1]}d{c[2]}p{c[3]}{c[4]}-" + "-".join(f"{k}by{len(m)}" for k, m in c[5])[:40]


@pytest.mark.parametrize("case", CASES, ids=name)
def test_attend(gpu, case):  # noqa: F811
    H, G, D, P, dtype, runs = case
    rng = np.random.default_rng(21)
    table, kv, ql, pages = layout(rng, runs, P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP[dtype])
    got = attend(gpu, codes, exps, table, kv, ql, q, dtype, runs=sum(k > 0 for k, _ in runs))
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    assert ref.close(got, want, bound, dtype)


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
@pytest.mark.parametrize("case", [CASES[1], CASES[9]], ids=name)
def test_scales(gpu, case, scale):  # noqa: F811
    """No scale (all keys alike), a negative one, and one that leaves one key."""
    H, G, D, P, dtype, runs = case
    rng = np.random.default_rng(22)
    table, kv, ql, pages = layout(rng, runs, P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP[dtype])
    got = attend(gpu, codes, exps, table, kv, ql, q, dtype, scale=scale)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), scale)
    assert ref.close(got, want, bound, dtype)


@pytest.mark.parametrize("case", [CASES[1], CASES[6]], ids=name)
def test_windows_and_long_sequences(gpu, case):  # noqa: F811
    """Calls that share nothing in a batch made to share: the same bits as in one
    that was not."""
    H, G, D, P, dtype, runs = case
    rng = np.random.default_rng(23)
    table, kv, ql, pages = layout(rng, runs, P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP[dtype])
    for kw in ({"window": 100}, {"window": 30, "sinks": 70}):
        both = [attend(gpu, codes, exps, table, kv, ql, q, dtype, shared, **kw) for shared in (True, False)]
        assert both[0].tobytes() == both[1].tobytes()
    many = np.concatenate([q] * 16, 1)                   # more than 32 rows of a kv head
    both = [attend(gpu, codes, exps, table, kv, ql, many, dtype, shared) for shared in (True, False)]
    assert both[0].tobytes() == both[1].tobytes()


@pytest.mark.parametrize("case", [CASES[1], CASES[6]], ids=name)
def test_values_that_are_not_finite(gpu, case):  # noqa: F811
    """NaN values of a shared page reach every row, own pages' only their
    sequence's, hidden ones none; NaN keys are NaN for all rows that see them."""
    H, G, D, P, dtype, runs = case
    rng = np.random.default_rng(24)
    table, kv, ql, pages = layout(rng, runs, P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    codes[table[0][1], 1, 0, 5, 7] = 0x7f                # shared value, head 0
    codes[table[1][kv[1] // P if kv[1] % P else kv[1] // P - 1], 1, 1, (kv[1] - 1) % P, 3] = 0xff   # own value, head 1
    last = table[2][(kv[2] - 1) // P]
    codes[last, :, :, (kv[2] - 1) % P + 1:] = 0x7f       # behind the last key
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP[dtype])
    got = attend(gpu, codes, exps, table, kv, ql, q, dtype)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    assert np.isnan(want[:, :G, 7]).all() and np.isnan(want[1, G:2 * G, 3]).all() and np.isnan(want).mean() < 0.1
    assert ref.close(got, want, np.nan_to_num(bound), dtype)
    # a query of infinities and one of NaN leave the other sequences alone
    q[0, 0, 0], q[1, 0, 0] = np.inf, np.nan
    again = attend(gpu, codes, exps, table, kv, ql, q, dtype)
    keep = np.ones(q.shape[:2], bool)
    keep[:2, 0] = False
    assert ref.close(again[keep], want[keep], np.nan_to_num(bound)[keep], dtype)


def test_uneven_pages(gpu):  # noqa: F811
    """Page exponents far apart between shared and own keys, values of 2^60."""
    rng = np.random.default_rng(25)
    H, G, D, P = 1, 4, 64, 64
    for members in (3, 20):
        table, kv, ql, pages = layout(rng, [(256, [(40, 1)] * members)], P)
        codes, exps = ref.pool(rng, pages, H, P, D)
        exps[:, 1] = rng.integers(-32, 55, exps[:, 1].shape)
        exps[:, 0] = rng.integers(-8, -2, exps[:, 0].shape)
        q = rng.standard_normal((members, H * G, D)).astype(np.float16)
        got = attend(gpu, codes, exps, table, kv, ql, (q * 0.1).astype(NP["bf16"]), "bf16")
        want, bound = ref.attend(codes, exps, table, kv, ql, (q * 0.1).astype(NP["bf16"]).astype(np.float64), D ** -0.5)
        assert ref.close(got, want, bound, "bf16")


def test_update_and_graph(gpu):  # noqa: F811
    """A captured call replays with other lengths, runs and pages: fewer, more and
    longer runs than the batch was made for among them."""
    import torch
    rng = np.random.default_rng(26)
    H, G, D, P = 2, 4, 64, 64
    made = [(256, [(30, 1)] * 12), (128, [(5, 1)] * 4)]
    other = [[(64, [(3, 1)] * 16)], [(128, [(5, 1)] * 4), (128, [(64, 1)] * 4), (128, [(2, 1)] * 4), (64, [(9, 1)] * 4)],
             [(0, [(100 + i, 1)]) for i in range(16)], [(256, [(1 + 2 * i, 1) for i in range(15)]), (0, [(1, 0)])], made]
    pages = 80
    codes, exps = ref.pool(rng, pages, H, P, D)
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    table, kv, ql, used = layout(rng, made, P)
    width = 8

    def wide(t):
        return np.concatenate([t, np.zeros((len(t), width - t.shape[1]), np.int32)], 1)
    side = torch.cuda.Stream()
    batch = cache.batch(wide(table), kv, ql, stream=side, shared=True)
    assert batch._s.max_runs == 2 and batch._s.max_tokens == 12
    q = torch.randn((16, H * G, D), device="cuda").half()
    out = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    batch.reserve(H * G, stream=side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        batch.attend(0, q, out, stream=side)
    for runs in other:
        table, kv, ql, used = layout(rng, runs, P)
        assert used <= pages
        q.copy_(torch.randn_like(q))
        batch.update(wide(table), kv, ql, stream=side)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out.zero_()
            graph.replay()
        batch.check_errors(stream=side)
        n = sum(ql)
        want, bound = ref.attend(codes, exps, table, kv, ql, q.double().cpu().numpy()[:n], D ** -0.5)
        assert ref.close(out.cpu().numpy()[:n], want, bound, "f16")
        assert (out[n:] == 0).all()
    torch.cuda.synchronize()
    del graph
    batch.close()


def test_runs_that_cannot_be(gpu):  # noqa: F811
    """What the device arrays might say when their owner overwrites them: each
    such run's sequences are attended to by themselves or skipped and reported,
    the others as ever."""
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(27)
    H, G, D, P = 1, 4, 64, 64
    runs = [(128, [(30, 1)] * 3), (192, [(5, 1)] * 12)]
    table, kv, ql, pages = layout(rng, runs, P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    q = rng.standard_normal((15, H * G, D)).astype(np.float16)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    good = np.zeros((3, 15), np.int32)
    good[0] = [0] * 3 + [3] * 12
    good[1], good[1, 0], good[1, 3] = 1, 3, 12
    good[2] = [128] * 3 + [192] * 12
    for spot, value, hit, reported in [
            (None, 0, 0, False), ((1, 0), 99, 3, True), ((2, 0), 100, 3, True), ((2, 0), 64 * 99, 3, True),
            ((2, 0), 192, 3, True), ((2, 0), -64, 3, True), ((0, 1), 5, 1, False), ((0, 1), -7, 1, False),
            ((0, 1), 2, 1, False), ((1, 3), 2, 12, False), ((1, 0), -5, 3, False), ((0, 0), 1, 3, False),
            ((1, 0), 15, 15, None)]:
        batch = cache.batch(table, kv, ql, shared=True)
        batch.reserve(H * G)
        said = good.copy()
        if spot is not None:
            said[spot] = value
        gpu.dev.htod(batch._s.runs, said)
        batch._plan((H * G, 0, 0), gpu.dev.stream)
        out = gpu.put(np.full(q.shape, 77).astype(np.float16), "f16")
        batch.attend(0, gpu.put(q, "f16"), out)
        got = gpu.get(out, q.shape, np.float16)
        if reported:
            with pytest.raises(EmmyError, match="longer than its row"):
                batch.check_errors()
        elif reported is False:
            batch.check_errors()
        left = (got == 77).all((1, 2))
        right = np.array([left[i] or ref.close(got[i:i + 1], want[i:i + 1], bound[i:i + 1], "f16") for i in range(15)])
        assert right[hit:].all() and not left[hit:].any()
        if reported is False:
            assert right.all() and not left.any()
        batch.close()
    # a plan for the one kind of call is not for the other
    plain, shared = cache.batch(table, kv, ql), cache.batch(table, kv, ql, shared=True)
    for b in (plain, shared):
        b.reserve(H * G)
    for a, b in ((plain, shared), (shared, plain)):
        a._ws = b._ws = max(a._ws, b._ws, key=lambda w: w[1])
        kept = a._plans[H * G, 0, 0]
        a._plans[H * G, 0, 0] = (b._plans[H * G, 0, 0][0], max(kept[1], b._plans[H * G, 0, 0][1]))
        if b._plans[H * G, 0, 0][1] >= kept[1]:
            out = gpu.put(np.full(q.shape, 77).astype(np.float16), "f16")
            a.attend(0, gpu.put(q, "f16"), out)
            with pytest.raises(EmmyError, match="another call"):
                a.check_errors()
            assert (gpu.get(out, q.shape, np.float16) == 77).all()
        a._plans[H * G, 0, 0] = kept


@pytest.mark.parametrize("group,seqs", [(4, 8), (8, 40)], ids=["rows", "tiles"])
def test_runs_that_overlap(gpu, group, seqs):  # noqa: F811
    """Device arrays that make each sequence the first of a run of all behind it: more
    rows than a call has room for, so nothing is shared, and that is reported."""
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(33)
    H, D, P = 2, 64, 64
    table, kv, ql, pages = layout(rng, [(192, [(1 + i, 1) for i in range(seqs)])], P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    q = rng.standard_normal((seqs, H * group, D)).astype(np.float16)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    batch = cache.batch(table, kv, ql, shared=True)
    batch._s.max_runs = seqs
    batch.reserve(H * group)
    each = np.arange(seqs)
    gpu.dev.htod(batch._s.runs, np.stack([each, seqs - each, 0 * each + 192]).astype(np.int32))
    batch._plan((H * group, 0, 0), gpu.dev.stream)
    out = gpu.put(np.zeros_like(q), "f16")
    batch.attend(0, gpu.put(q, "f16"), out)
    assert ref.close(gpu.get(out, q.shape, np.float16), want, bound, "f16")
    with pytest.raises(EmmyError, match="longer than its row"):
        batch.check_errors()
    batch.close()


@pytest.mark.parametrize("group,seqs", [(4, 4), (8, 20)], ids=["rows", "tiles"])
def test_lengths_that_change_after_the_plan(gpu, group, seqs):  # noqa: F811
    """A plan computes the rows of the lengths that it was made from."""
    rng = np.random.default_rng(34)
    H, D, P = 1, 128, 64
    table, kv, ql, pages = layout(rng, [(256, [(2 + 3 * i, 1 + i % 2) for i in range(seqs)])], P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    q = rng.standard_normal((sum(ql), H * group, D)).astype(np.float16)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    batch = cache.batch(table, kv, ql, shared=True)
    batch.reserve(H * group)
    # the first ones' tokens are another's: none of the even ones, two of each odd one
    starts = np.concatenate([[0], np.cumsum([2 * (i % 2) for i in range(seqs)])]).astype(np.int32)
    gpu.dev.htod(batch._d.q_starts, starts)
    out = gpu.put(np.zeros_like(q), "f16")
    batch.attend(0, gpu.put(q, "f16"), out)
    batch.check_errors()
    assert ref.close(gpu.get(out, q.shape, np.float16), want, bound, "f16")
    batch.close()


def test_more_runs_than_there_is_room_for(gpu):  # noqa: F811
    """Device arrays that name more runs, or longer ones, than the call was made for:
    those beyond are attended to by themselves."""
    rng = np.random.default_rng(29)
    H, G, D, P = 2, 4, 128, 64
    for sizes in ((4, 4, 4), (12, 12, 12)):              # row kernel, tile kernel
        runs = [(128, [(30 + i, 1) for i in range(n)]) for n in sizes]
        table, kv, ql, pages = layout(rng, runs, P)
        codes, exps = ref.pool(rng, pages, H, P, D)
        cache, _, _ = cache_of(gpu, codes[None], exps[None])
        T = len(kv)
        q = rng.standard_normal((T, H * G, D)).astype(np.float16)
        want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
        for max_runs, max_tokens in ((1, sizes[0]), (2, sizes[0]), (3, sizes[0] - 1), (3, T)):
            batch = cache.batch(table, kv, ql, shared=True)
            batch._s.max_runs, batch._s.max_tokens = max_runs, max_tokens
            out = gpu.put(np.zeros_like(q), "f16")
            batch.attend(0, gpu.put(q, "f16"), out)
            batch.check_errors()
            assert ref.close(gpu.get(out, q.shape, np.float16), want, bound, "f16")
            batch.close()


def test_most_sequences(gpu):  # noqa: F811
    """4096 sequences in one run, and in 1024 of four."""
    rng = np.random.default_rng(30)
    H, G, D, P, n = 1, 2, 64, 64, 4096
    codes, exps = ref.pool(rng, 1100, H, P, D)
    q = rng.standard_normal((n, H * G, D)).astype(np.float16)
    kv = [64 + 1 + i % 5 for i in range(n)]
    for members in (n, 4):
        table = np.stack([np.arange(n) // members % 1024, 1024 + np.arange(n) % 70], 1).astype(np.int32)
        got = attend(gpu, codes, exps, table, kv, [1] * n, q, "f16", runs=n // members)
        some = rng.integers(0, n, 64)
        want, bound = ref.attend(codes, exps, table[some], [kv[i] for i in some], [1] * 64, q[some].astype(np.float64), D ** -0.5)
        assert ref.close(got[some], want, bound, "f16")


def test_streams_and_slices(gpu):  # noqa: F811
    """On a stream that is not the batch's own; q and out slices of one array; layers."""
    import torch
    rng = np.random.default_rng(31)
    H, G, D, P, dtype, runs = CASES[6]
    table, kv, ql, pages = layout(rng, runs, P)
    both = [ref.pool(rng, pages, H, P, D) for _ in range(2)]
    cache, _, _ = cache_of(gpu, np.stack([c for c, _ in both]), np.stack([e for _, e in both]))
    batch = cache.batch(table, kv, ql, shared=True)
    x = torch.randn((len(ql), 2 * H * G, D), device="cuda").bfloat16()
    torch.cuda.synchronize()
    q, out = x[:, :H * G], x[:, H * G:]
    side = torch.cuda.Stream()
    for layer, (codes, exps) in enumerate(both):
        batch.attend(layer, q, out, stream=side)
        batch.check_errors(stream=side)
        want, bound = ref.attend(codes, exps, table, kv, ql, q.double().cpu().numpy(), D ** -0.5)
        assert ref.close(out.float().cpu().numpy(), want, bound, dtype)
    batch.close()


def test_forks_generate_together(gpu):  # noqa: F811
    """A prompt, forks of it, and steps of all of them at once: rotated appends and
    shared attention, against the same in 64 bits over what the cache holds."""
    import torch
    from ptxgen import KVCache, KVSequences, Rotary
    from tests import rotary_oracle
    H, G, D, n, forks, steps = 2, 4, 64, 200, 20, 3
    st = torch.cuda.current_stream().cuda_stream
    codes = torch.zeros((2, 120, 2, H, 64, D), dtype=torch.uint8, device="cuda")
    exps = torch.zeros((2, 120, 2, H), dtype=torch.int8, device="cuda")
    cache = KVCache(120, H, D, layers=2, storage=(codes, exps))
    seqs, rot = KVSequences(cache), Rotary(D, dims=32, interleaved=True)
    root = seqs.new()

    def step(ids, counts, shared):
        batch = seqs.batch(ids, counts, stream=st, shared=shared)
        T = sum(counts)
        x = torch.randn((T, H * G + 2 * H, D), device="cuda").bfloat16()
        place = np.concatenate([np.arange(seqs.length(s) - c, seqs.length(s)) for s, c in zip(ids, counts)])
        for layer in range(2):
            q, out = torch.empty((T, H * G, D), device="cuda", dtype=torch.bfloat16), torch.empty((T, H * G, D), device="cuda", dtype=torch.bfloat16)
            batch.append(layer, x[:, H * G:H * G + H], x[:, H * G + H:], stream=st, rotary=rot, q=x[:, :H * G], q_out=q)
            batch.attend(layer, q, out, stream=st)
            batch.check_errors(stream=st)
            want_q, bq = rotary_oracle.rotate(rot, x[:, :H * G].double().cpu().numpy(), place, to="16")
            assert rotary_oracle.close(q.double().cpu().numpy(), want_q, bq, "bf16")
            want, bound = ref.attend(codes[layer].cpu().numpy(), exps[layer].cpu().numpy(), seqs.table(ids).tolist(),
                                     [seqs.length(s) for s in ids], counts, q.double().cpu().numpy(), D ** -0.5)
            assert ref.close(out.float().cpu().numpy(), want, bound, "bf16")
        return batch
    step([root], [n], False)
    ids = [root] + [seqs.fork(root) for _ in range(forks - 1)]
    for i in range(steps):
        batch = step(ids, [1 + (i == 1) * (j % 3) for j in range(forks)], True)
        assert batch._s.max_runs == 1
    assert seqs.pages(ids[0])[:n // 64] == seqs.pages(ids[7])[:n // 64]
    cache.close()


@pytest.mark.parametrize("case", [CASES[1], CASES[6], CASES[14]], ids=name)
def test_waits_that_run_out(gpu, case):  # noqa: F811
    """Blocks that withhold their own first keys: reported, and the batch then
    computes as if nothing had been."""
    from ptxgen.kvcache import WORKSPACE_ZERO
    from ptxgen.runtime import EmmyError, load_library
    H, G, D, P, dtype, runs = case
    rng = np.random.default_rng(28)
    table, kv, ql, pages = layout(rng, runs, P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP[dtype])
    qd, od = gpu.put(q, dtype), gpu.put(np.zeros_like(q), dtype)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    batch, L = cache.batch(table, kv, ql, shared=True), load_library()
    for stall in (1, 2, 3):
        L.emmy_kv8_wait_limit(1000000, stall)
        try:
            batch.attend(0, qd, od)
        finally:
            L.emmy_kv8_wait_limit(2000000000, 0)
        with pytest.raises(EmmyError, match="0x403"):
            batch.check_errors()
        counters = np.empty(WORKSPACE_ZERO, np.uint8)
        gpu.dev.dtoh(counters, batch._ws[0])
        gpu.dev.sync()
        assert not counters.any()
        batch.attend(0, qd, od)
        batch.check_errors()
        assert ref.close(gpu.get(od, q.shape, NP[dtype]), want, bound, dtype)
    batch.close()


@pytest.mark.parametrize("group,members", [(4, 4), (8, 12)], ids=["rows", "tiles"])
@pytest.mark.parametrize("field,value", [("max_runs", 1), ("max_runs", 2), ("max_tokens", 1), ("tokens", -1)])
def test_plan_of_another_layout(gpu, group, members, field, value):  # noqa: F811
    """A plan that was made for other runs or tokens lies elsewhere in the same bytes:
    refused or reported, nothing written, and no harm to the next call."""
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(35)
    H, D, P = 2, 64, 64
    runs = [(128, [(70, 2)] * members), (64, [(9, 1)] * members), (192, [(5, 1)] * members)]
    table, kv, ql, pages = layout(rng, runs, P)
    codes, exps = ref.pool(rng, pages, H, P, D)
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    q = rng.standard_normal((sum(ql), H * group, D)).astype(np.float16)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    batch = cache.batch(table, kv, ql, shared=True)
    assert (batch._s.max_runs, batch._s.max_tokens, batch.max_q) == (3, 2 * members, 2)
    batch.reserve(H * group)
    made = (batch._s.max_runs, batch._s.max_tokens, batch._d.tokens)
    where = batch._s if field in ("max_runs", "max_tokens") else batch._d
    setattr(where, field, getattr(where, field) + value if value < 0 else value)
    import ctypes
    ws, plan = ctypes.c_uint64(), ctypes.c_uint64()
    assert batch.L.emmy_kv8_attend_shared_sizes(batch._ref, batch._sref, H * group, ctypes.byref(ws), ctypes.byref(plan)) == 0
    at, held = batch._plans[H * group, 0, 0]
    out = gpu.put(np.full(q.shape, 77).astype(np.float16), "f16")
    if plan.value > held or ws.value > batch._ws[1]:     # the host knows already
        assert (group, field) == (8, "max_tokens")
        with pytest.raises(EmmyError, match="too small"):
            batch.attend(0, gpu.put(q, "f16"), out)
    else:
        batch.attend(0, gpu.put(q, "f16"), out)
        with pytest.raises(EmmyError, match="another call"):
            batch.check_errors()
    assert (gpu.get(out, q.shape, np.float16) == 77).all()
    batch._s.max_runs, batch._s.max_tokens, batch._d.tokens = made       # as it was made
    batch.attend(0, gpu.put(q, "f16"), out)
    batch.check_errors()
    assert ref.close(gpu.get(out, q.shape, np.float16), want, bound, "f16")
    batch.close()


@pytest.mark.parametrize("lens,ql,field,value", [
    # 500 sequences of 20 rows of a kv head are 1000 blocks of rows, of 16 rows 500
    ([200] * 500, [5] * 500, "max_q", 4),
    # 500 tokens of 4 heads are 7 + 2 units of 256 rows at most, 400 are 6 + 2
    ([300, 300], [300, 200], "tokens", 400),
], ids=["rows", "tiles"])
def test_plan_of_another_layout_unshared(gpu, lens, ql, field, value):  # noqa: F811
    """The same of calls that share nothing."""
    import ctypes
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(36)
    H, G, D, P = 1, 4, 64, 64
    width = -(-max(lens) // P)
    table = np.arange(width * len(lens)).reshape(len(lens), width)
    codes, exps = ref.pool(rng, table.size, H, P, D)
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    q = rng.standard_normal((sum(ql), H * G, D)).astype(np.float16)
    batch = cache.batch(table, lens, ql)
    batch.reserve(H * G)
    setattr(batch._d, field, value)
    ws, plan = ctypes.c_uint64(), ctypes.c_uint64()
    assert batch.L.emmy_kv8_attend_sizes(batch._ref, H * G, ctypes.byref(ws), ctypes.byref(plan)) == 0
    assert plan.value < batch._plans[H * G, 0, 0][1] and ws.value <= batch._ws[1]
    out = gpu.put(np.full(q.shape, 77).astype(np.float16), "f16")
    batch.attend(0, gpu.put(q, "f16"), out)
    with pytest.raises(EmmyError, match="another call"):
        batch.check_errors()
    assert (gpu.get(out, q.shape, np.float16) == 77).all()
    batch.close()


@pytest.mark.parametrize("heads,head_dim,dtype", [(160, 128, "bf16"), (320, 64, "f16")])
def test_more_units_than_blocks(gpu, heads, head_dim, dtype):  # noqa: F811
    """A run's 40 rows of each of many kv heads: blocks of the tile kernel take two or
    three units one after another."""
    rng = np.random.default_rng(37)
    table, kv, ql, pages = layout(rng, [(640, [(3 + 40 * i, 1) for i in range(5)])], 64)
    codes, exps = ref.pool(rng, pages, heads, 64, head_dim)
    q = rng.standard_normal((5, heads * 8, head_dim)).astype(NP[dtype])
    got = attend(gpu, codes, exps, table, kv, ql, q, dtype, runs=1)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), head_dim ** -0.5)
    assert ref.close(got, want, bound, dtype)
