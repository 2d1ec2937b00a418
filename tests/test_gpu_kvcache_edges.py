"""The paged 8-bit cache where its arithmetic ends: scores past f32's whole
numbers and near the end of its range; streams that share a handle;
segments of more parts than one level of joins takes, the largest pages of f32."""

import threading

import ml_dtypes
import numpy as np
import pytest

from tests import kv8_oracle as ref
from tests.test_gpu_kvcache import NP, attend_gpu, cache_of, gpu  # noqa: F401 - a fixture

pytestmark = pytest.mark.gpu


def filled(pages, D, keys, values, P=64):
    """Codes and exponents of one head whose key j is keys[j] (code, exponent)
    in its first element, zeros elsewhere, and whose value j is values[j]
    (element, number that e4m3 holds); a page has one exponent for its keys."""
    codes, exps = np.zeros((pages, 2, 1, P, D), np.uint8), np.zeros((pages, 2, 1), np.int8)
    for j, (number, e) in keys.items():
        codes[j // P, 0, 0, j % P, 0] = ref.encode(number)
        exps[j // P, 0, 0] = e
    for j, (d, number) in values.items():
        codes[j // P, 1, 0, j % P, d] = ref.encode(number)
    return codes, exps


def log2_score(D, scale, q, number, e):
    return (D ** -0.5 if scale is None else scale) * np.log2(np.e) * q * number * 2.0 ** e


# K of the two keys in units of 2^6: scores below and above 2^27, whose ratio is
# less than the scale's over its power of two
@pytest.mark.parametrize("D,scale,small,large", [(64, None, 352, 384), (128, 0.17, 256, 288)])
@pytest.mark.parametrize("first", ["small", "large"])
@pytest.mark.parametrize("L,n,at", [
    (200, 100, (5, 70)),            # one unit, two of its chunks
    (3000, 40, (130, 2500)),        # two parts of a unit cut along its keys
    (300, 1, (5, 150)),             # the row kernel
])
def test_a_maximum_that_crosses_whole_numbers(gpu, D, scale, small, large, first, L, n, at):  # noqa: F811
    """Of two keys with scores of 2^27 and less and of 2^27 and more, 10^7
    apart, the larger takes all: the output is its value, exactly."""
    q = 2.0 ** 15
    a, b = (log2_score(D, scale, q, k, 6) for k in (small, large))
    assert 1.2e8 < a < 2.0 ** 27 < b < 1.6e8 and b - a > 1e7
    keys = {at[0]: (small, 6), at[1]: (large, 6)} if first == "small" else {at[0]: (large, 6), at[1]: (small, 6)}
    winner = at[1] if first == "small" else at[0]
    values = {j: (0, 2.0 if j == winner else 1.0) for j in at}
    pages = -(-L // 64)
    codes, exps = filled(pages, D, keys, values)
    rows = np.zeros((n, 1, D), np.float16)
    rows[:, :, 0] = q
    got = attend_gpu(gpu, codes, exps, np.arange(pages, dtype=np.int32)[None], [L], [n], rows, "f16", scale=scale)
    assert (got[:, 0, 0] == 2.0).all() and not got[:, 0, 1:].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L,n,low,at", [
    (200, 100, range(64), (70, 90)),                    # a first chunk far below the next
    (3000, 40, range(64, 3000), (10, 20)),              # later parts of a cut unit far below the first
    (200, 2, range(64), (70, 90)),
])
def test_scores_far_below_the_others(gpu, D, L, n, low, at):  # noqa: F811
    """Chunks of scores of -1.4e8 leave the weights of two ordinary keys as
    they are: exp(s0 - s1) over their sum."""
    q = 2.0 ** 15
    keys = {j: (-256.0 if (j // 64) * 64 in low else -448.0, 7 if (j // 64) * 64 in low else -12) for j in range(L)}
    keys[at[0]], keys[at[1]] = (10.0, -12), (11.0, -12)
    assert log2_score(D, 0.125, q, -256.0, 7) < -2.0 ** 27
    pages = -(-L // 64)
    codes, exps = filled(pages, D, keys, {at[0]: (0, 1.0), at[1]: (1, 1.0)})
    rows = np.zeros((n, 1, D), np.float16)
    rows[:, :, 0] = q
    got = attend_gpu(gpu, codes, exps, np.arange(pages, dtype=np.int32)[None], [L], [n], rows, "f16", scale=0.125)
    w = np.exp(-0.125 * q * 2.0 ** -12)
    want = np.zeros(D)
    want[:2] = w / (1 + w), 1 / (1 + w)
    # the other keys' weights are below 2^-600; weights and output are f16, and a
    # score of 16 in log2 units is rounded by 2^-20 at most, which moves a weight by ln 2 of that
    tol = want * (2 * 2.0 ** -11 + 2.0 ** -18)
    assert (np.abs(got[:, 0].astype(float) - want) <= tol).all()


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("window", [1, 2])
def test_scores_near_the_end_of_f32(gpu, n, window):  # noqa: F811
    """Every visible key has a score of -2^105 and less, far below -1e30: a
    row that sees one key is its value, one that sees two the larger's."""
    D, L, q = 64, 130, 2.0 ** 90
    rng = np.random.default_rng(4)
    pages = 3
    codes, exps = filled(pages, D, {j: (-448.0 if j % 2 else -224.0, 10) for j in range(L)}, {})
    codes[:, 1, 0] = ref.encode(rng.standard_normal((pages, 64, D)) * 10)
    assert -3.4e38 < log2_score(D, None, q, -448.0, 10) < log2_score(D, None, q, -224.0, 10) < -1e31
    rows = np.zeros((n, 1, D), ml_dtypes.bfloat16)
    rows[:, :, 0] = q
    table = np.arange(pages, dtype=np.int32)[None]
    got = attend_gpu(gpu, codes, exps, table, [L], [n], rows, "bf16", window=window)
    _, v = ref.held(codes, exps, table, 0, L, 0)
    for i in range(n):
        p = L - n + i
        key = p if window == 1 or p % 2 == 0 else p - 1
        assert (got[i, 0].astype(float) == v[key]).all()       # e4m3 is exact in bf16


def test_threads_on_their_default_streams():
    """One handle, a stream for each thread: batches made and closed one after
    another in each, with work still queued."""
    torch = pytest.importorskip("torch")
    from ptxgen import KVCache
    rng = np.random.default_rng(5)
    P, D, H, kv, ql = 64, 64, 1, [900, 70, 300], [1, 2, 1]
    codes, exps = ref.pool(rng, 24, H, P, D)
    table = ref.tables(rng, 24, kv, P)
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache = KVCache(24, H, D, storage=(c, e))
    q = torch.from_numpy(rng.standard_normal((4, 2, D))).half().cuda()
    outs, failed = [torch.zeros_like(q) for _ in range(4)], []
    torch.cuda.synchronize()

    def work(i):
        try:
            pick = [0, 1, 2] if i % 2 else [2, 0, 1]                    # unlike tables and lengths
            rows = torch.cat([q[sum(ql[:b]):sum(ql[:b + 1])] for b in pick])
            torch.cuda.synchronize()
            for _ in range(20):
                batch = cache.batch(table[pick], [kv[b] for b in pick], [ql[b] for b in pick], stream=2)
                batch.attend(0, rows, outs[i], stream=2)
                batch.close()
            batch = cache.batch(table[pick], [kv[b] for b in pick], [ql[b] for b in pick], stream=2)
            batch.check_errors(stream=2)                                # waits for the stream
            want, bound = ref.attend(codes, exps, table[pick], [kv[b] for b in pick], [ql[b] for b in pick],
                                     rows.cpu().numpy().astype(float), D ** -0.5)
            assert ref.close(outs[i].cpu().numpy(), want, bound, "f16")
        except BaseException as exc:  # noqa: BLE001 - reported below
            failed.append(exc)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed


def test_a_batch_that_goes_while_its_graph_runs():
    """Captured on the batch's own stream, replayed on another, dropped while
    replays are queued there: the next batches on its stream have other memory."""
    torch = pytest.importorskip("torch")
    from ptxgen import KVCache
    rng = np.random.default_rng(6)
    P, D, H, kv = 64, 64, 1, [3000, 500]
    codes, exps = ref.pool(rng, 60, H, P, D)
    table = ref.tables(rng, 60, kv, P)
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache = KVCache(60, H, D, storage=(c, e))
    q = torch.from_numpy(rng.standard_normal((2, 2, D))).half().cuda()
    out, other = torch.zeros_like(q), torch.zeros_like(q)
    st, elsewhere = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    batch = cache.batch(table, kv, stream=st)
    batch.reserve(2, stream=st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        for _ in range(50):
            batch.attend(0, q, out, stream=st)
    with torch.cuda.stream(elsewhere):
        for _ in range(10):
            graph.replay()
    del batch
    for _ in range(5):
        b = cache.batch([[0] * 47], [47 * P], [1], stream=st)          # other lengths, over the same sizes
        b.attend(0, q, other, stream=st)
        del b
    torch.cuda.synchronize()
    want, bound = ref.attend(codes, exps, table, kv, [1, 1], q.cpu().numpy().astype(float), D ** -0.5)
    assert ref.close(out.cpu().numpy(), want, bound, "f16")


@pytest.mark.parametrize("prompts,singles", [([300, 90], 40), ([64], 300)])
def test_prompts_beside_single_tokens_right_behind_append(prompts, singles):
    """Both kernels of the call read what the append right before it wrote."""
    torch = pytest.importorskip("torch")
    from ptxgen import KVCache
    rng = np.random.default_rng(8)
    P, D, H, G = 64, 128, 2, 2
    ql = prompts + [1] * singles
    kv = [n + int(rng.integers(0, 200)) for n in prompts] + rng.integers(1, 500, singles).tolist()
    pages = sum(-(-n // P) for n in kv)
    codes, exps = ref.pool(rng, pages, H, P, D)
    table = ref.tables(rng, pages, kv, P)
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache = KVCache(pages, H, D, storage=(c, e))
    n = sum(ql)
    k, v = (rng.standard_normal((2, n, H, D)) * 4).astype(np.float16)
    q = torch.from_numpy(rng.standard_normal((n, H * G, D))).half().cuda()
    kd, vd, c0, e0 = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), c.clone(), e.clone()
    st = torch.cuda.current_stream()
    batch, outs = cache.batch(table, kv, ql, stream=st), []
    for _ in range(10):
        c.copy_(c0)
        e.copy_(e0)
        outs.append(torch.empty_like(q))
        batch.append(0, kd, vd, stream=st)
        batch.attend(0, q, outs[-1], stream=st)
    batch.check_errors(stream=st)
    after = ref.append(codes, exps, table, kv, ql, k.astype(float), v.astype(float))
    assert (c[0].cpu().numpy() == after[0]).all() and (e[0].cpu().numpy() == after[1]).all()
    want, bound = ref.attend(*after, table, kv, ql, q.cpu().numpy().astype(float), D ** -0.5)
    assert ref.close(outs[0].cpu().numpy(), want, bound, "f16")
    assert all(torch.equal(o, outs[0]) for o in outs)
    counters = torch.empty(16384, dtype=torch.uint8)
    cache.dev.dtoh(counters.numpy(), batch._ws[0])
    cache.dev.sync()
    assert not counters.any()


@pytest.mark.parametrize("H,G,D,dtype,seqs", [
    (1, 8, 128, "bf16", [(70000, 1)]),                         # clusters of four, 28 results
    (2, 2, 64, "f16", [(131071, 2)]),                          # 47
    (1, 3, 64, "bf16", [(45001, 1)] + [(200 + i, 1) for i in range(60)]),      # single parts, more than 200
])
def test_joins_of_two_levels(gpu, H, G, D, dtype, seqs):  # noqa: F811
    """Segments with more results than one CTA joins at once."""
    rng = np.random.default_rng(H + G)
    P = 64
    kv, ql = [a for a, _ in seqs], [b for _, b in seqs]
    pages = sum(-(-n // P) for n in kv)
    codes, exps = ref.pool(rng, pages, H, P, D)
    table = ref.tables(rng, pages, kv, P)
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP[dtype])
    got = attend_gpu(gpu, codes, exps, table, kv, ql, q, dtype)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(np.float64), D ** -0.5)
    assert ref.close(got, want, bound, dtype)


@pytest.mark.parametrize("H,dtype,seqs", [(2, "f32", [(600, 345), (257, 2)]), (1, "f32", [(256, 256), (300, 44)])])
def test_append_pages_of_one_buffer(gpu, H, dtype, seqs):  # noqa: F811
    """f32 pages of 256 tokens and 128 elements fill the shared memory: one
    buffer, one (side, head) a CTA."""
    rng = np.random.default_rng(H)
    P, D = 256, 128
    kv, ql = [a for a, _ in seqs], [b for _, b in seqs]
    pages = sum(-(-n // P) for n in kv) + 1
    codes, exps = ref.pool(rng, pages, H, P, D)
    table = ref.tables(rng, pages, kv, P)
    x = rng.standard_normal((2, sum(ql), H, D)) * 2.0 ** rng.integers(-6, 7, (2, sum(ql), H, 1))
    x = x.astype(NP[dtype])
    cache, cd, ed = cache_of(gpu, codes[None], exps[None])
    batch = cache.batch(table, kv, ql)
    batch.append(0, gpu.put(x[0], dtype), gpu.put(x[1], dtype))
    batch.check_errors()
    want = ref.append(codes, exps, table, kv, ql, x[0].astype(float), x[1].astype(float))
    assert (gpu.get(ed, exps.shape, np.int8) == want[1]).all()
    assert (gpu.get(cd, codes.shape, np.uint8) == want[0]).all()
    batch.close()


@pytest.mark.parametrize("n", [1, 40])
def test_exponents_outside_their_range(gpu, n):  # noqa: F811
    """Adopted storage may hold any int8: attend takes it for the range's end,
    as append does with a page that held tokens."""
    rng = np.random.default_rng(9)
    P, D, L = 64, 64, 64 * 4 + 30
    codes, exps = ref.pool(rng, 5, 1, P, D, spread=0.0)
    codes[:, 0] = 0                                           # every key alike
    table = ref.tables(rng, 5, [L], P)
    for odd in ([0, -128, 3, -33, 0], [64, 0, 127, 0, -128]):
        exps[:, 1, 0] = odd
        exps[:, 0, 0] = odd[::-1]
        q = rng.standard_normal((n, 2, D)).astype(ml_dtypes.bfloat16)
        got = attend_gpu(gpu, codes, exps, table, [L], [n], q, "bf16")
        kept = np.clip(exps, ref.E_MIN, ref.E_MAX)
        want, bound = ref.attend(codes, kept, table, [L], [n], q.astype(float), D ** -0.5)
        assert ref.close(got, want, bound, "bf16")


def test_q_and_out_as_slices_of_one_array():
    """Rows in turn do not overlap; rows that share an element do."""
    torch = pytest.importorskip("torch")
    from ptxgen import KVCache
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(10)
    P, D, H, G, kv, ql = 64, 64, 2, 2, [70, 300, 9], [1, 40, 2]
    codes, exps = ref.pool(rng, 8, H, P, D)
    table = ref.tables(rng, 8, kv, P)
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache, T, heads = KVCache(8, H, D, storage=(c, e)), sum(ql), H * G
    q0 = torch.from_numpy(rng.standard_normal((T, heads, D))).half().cuda()
    want, bound = ref.attend(codes, exps, table, kv, ql, q0.cpu().numpy().astype(float), D ** -0.5)
    batch = cache.batch(table, kv, ql, stream=0)
    wide = torch.zeros((T, 3 * heads, D), dtype=torch.float16, device="cuda")
    cols = torch.zeros((T, heads, 3 * D), dtype=torch.float16, device="cuda")
    deep = torch.zeros((heads, 3 * T, D), dtype=torch.float16, device="cuda")
    for q, out in ((wide[:, :heads], wide[:, 2 * heads:]), (wide[:, heads:2 * heads], wide[:, :heads]),
                   (cols[..., D:2 * D], cols[..., :D]), (cols[..., :D], cols[..., 2 * D:]),
                   (deep[:, :T].transpose(0, 1), deep[:, T:2 * T].transpose(0, 1))):
        q.copy_(q0)
        batch.attend(0, q, out, stream=0)
        assert ref.close(out.cpu().numpy(), want, bound, "f16") and torch.equal(q, q0)
    for q, out in ((wide[:, :heads], wide[:, heads - 1:2 * heads - 1]), (wide[:, 1:heads + 1], wide[:, :heads]),
                   (cols[..., :D], cols[..., D - 8:2 * D - 8]), (wide[:, :heads], wide[:, :heads]),
                   (deep[:, :T].transpose(0, 1), deep[:, T - 1:2 * T - 1].transpose(0, 1))):
        with pytest.raises(EmmyError, match="q and out overlap"):
            batch.attend(0, q, out, stream=0)
    batch.check_errors(stream=0)
