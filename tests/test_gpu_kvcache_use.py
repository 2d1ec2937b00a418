"""The paged 8-bit cache as programs use it: captured graphs, other streams,
threads, batches that reuse buffers, the largest counts, torch tensors."""

import threading

import numpy as np
import pytest

from tests import kv8_oracle as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def make(rng, kv, ql, H=2, G=4, D=128, P=64, extra=2, spread=3.0):
    """A filled cache over torch storage, its table and queries."""
    from ptxgen import KVCache
    pages = sum(-(-n // P) for n in kv) + extra
    codes, exps = ref.pool(rng, pages, H, P, D, spread=spread)
    table = ref.tables(rng, pages, kv, P)
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache = KVCache(pages, H, D, page_size=P, storage=(c, e))
    q = torch.from_numpy(rng.standard_normal((sum(ql), H * G, D))).half().cuda()
    return cache, codes, exps, table, q


def right(got, codes, exps, table, kv, ql, q, scale=None, **kw):
    want, bound = ref.attend(codes, exps, table, kv, ql, q.cpu().numpy().astype(float),
                             codes.shape[4] ** -0.5 if scale is None else scale, **kw)
    return ref.close(got.cpu().numpy(), want, bound, "f16")


def test_torch_tensors_on_their_stream():
    """The current torch stream, queries cut from a wider tensor."""
    rng = np.random.default_rng(0)
    kv, ql = [300, 70], [1, 3]
    cache, codes, exps, table, q = make(rng, kv, ql)
    wide = torch.zeros((4, 12, 128), dtype=torch.float16, device="cuda")
    wide[:, 2:10] = q
    out = torch.empty_like(q)
    st = torch.cuda.current_stream()
    batch = cache.batch(table, kv, ql, stream=st)
    got = batch.attend(0, wide[:, 2:10], out, stream=st)
    assert got is out and right(out, codes, exps, table, kv, ql, q)
    batch.check_errors(stream=st)


def test_two_captured_graphs_at_once_and_replay_after_update():
    """Each graph has a batch of its own; both replay at once on two streams
    many times; then new lengths go into one batch and its graph runs again."""
    rng = np.random.default_rng(1)
    sets = []
    for kv, ql in (([3000, 500], [1, 1]), ([900, 4000, 64], [3, 1, 2])):
        cache, codes, exps, table, q = make(rng, kv, ql)
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        batch = cache.batch(table, kv, ql, stream=st.cuda_stream)
        batch.reserve(q.shape[1], stream=st.cuda_stream)
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            for _ in range(5):
                batch.attend(0, q, out, stream=torch.cuda.current_stream())
        sets.append((kv, ql, cache, codes, exps, table, q, batch, out, graph, torch.cuda.Stream()))
    for _ in range(20):
        for s in sets:
            with torch.cuda.stream(s[-1]):
                s[-2].replay()
    torch.cuda.synchronize()
    for kv, ql, cache, codes, exps, table, q, batch, out, graph, st in sets:
        assert right(out, codes, exps, table, kv, ql, q)
        batch.check_errors(stream=0)
    kv, ql, cache, codes, exps, table, q, batch, out, graph, st = sets[0]
    shorter = [1200, 65]
    batch.update(table, shorter, [1, 1], stream=st)
    with torch.cuda.stream(st):
        graph.replay()
    torch.cuda.synchronize()
    assert right(out, codes, exps, table, shorter, [1, 1], q)
    batch.check_errors(stream=st)


def test_capture_on_a_stream_the_batch_never_saw():
    """Made and warmed up on the default stream, captured on another."""
    rng = np.random.default_rng(18)
    kv, ql = [3000, 500], [2, 1]
    cache, codes, exps, table, q = make(rng, kv, ql)
    batch, out = cache.batch(table, kv, ql, stream=0), torch.zeros_like(q)
    batch.attend(0, q, out, stream=0)
    torch.cuda.synchronize()
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.attend(0, q, out, stream=torch.cuda.current_stream())
    graph.replay()
    torch.cuda.synchronize()
    assert right(out, codes, exps, table, kv, ql, q)


def test_captured_step_appends_then_attends():
    """append and attend of one token in a graph, replayed as the sequence
    grows over a page's end."""
    from ptxgen import KVCache
    rng = np.random.default_rng(4)
    H, G, D, P = 1, 2, 64, 64
    codes, exps = ref.pool(rng, 4, H, P, D, spread=0.0)
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache = KVCache(4, H, D, storage=(c, e))
    table = np.array([[2, 0, 3]], np.int32)
    st = torch.cuda.Stream()
    k, v = (torch.zeros((1, H, D), dtype=torch.float16, device="cuda") for _ in range(2))
    q, out = (torch.zeros((1, H * G, D), dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    batch = cache.batch(table, [60], stream=st)
    batch.reserve(H * G, stream=st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        batch.append(0, k, v, stream=st)
        batch.attend(0, q, out, stream=st)
    for length in range(60, 70):
        x = rng.standard_normal((3, 1, H * G, D)).astype(np.float16) * 2.0 ** rng.integers(-3, 4)
        kk, vv, qq = x[0, :, :H], x[1, :, :H], x[2] / np.abs(x[2]).max()
        with torch.cuda.stream(st):
            for t, a in ((k, kk), (v, vv), (q, qq)):
                t.copy_(torch.from_numpy(a.astype(np.float16)))
        batch.update(table, [length], stream=st)
        with torch.cuda.stream(st):
            graph.replay()
        st.synchronize()
        codes, exps = ref.append(codes, exps, table, [length], [1], kk.astype(float), vv.astype(float))
        assert (c[0].cpu().numpy() == codes).all() and (e[0].cpu().numpy() == exps).all()
        assert right(out, codes, exps, table, [length], [1], q)


def test_threads_and_streams_of_their_own():
    """Four threads, each with a batch and a stream, on one cache."""
    rng = np.random.default_rng(2)
    kv, ql = [2000, 130, 64, 1], [1, 2, 1, 1]
    cache, codes, exps, table, q = make(rng, kv, ql)
    outs, failed = [torch.zeros_like(q) for _ in range(4)], []
    torch.cuda.synchronize()

    def work(i):
        try:
            st = torch.cuda.Stream()
            for _ in range(20):
                batch = cache.batch(table, kv, ql, stream=st)
                batch.attend(0, q, outs[i], window=0 if i % 2 else 100, stream=st)
                batch.close()
            st.synchronize()
        except Exception as exc:  # noqa: BLE001 - reported below
            failed.append(exc)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert right(out, codes, exps, table, kv, ql, q, window=0 if i % 2 else 100)


def test_batches_that_reuse_buffers_stay_right():
    """Batches made and dropped with work still queued, of changing sizes."""
    rng = np.random.default_rng(3)
    kv_all = [900, 30, 4000, 64, 129, 700]
    cache, codes, exps, table, q = make(rng, kv_all, [1] * 6)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for i in range(24):
        pick = rng.permutation(6)[:1 + i % 6]
        out = torch.zeros_like(q[:len(pick)])
        torch.cuda.synchronize() if i == 0 else None
        with torch.cuda.stream(st):
            qq = q[torch.from_numpy(pick).cuda()].contiguous()
        batch = cache.batch(table[pick], [kv_all[b] for b in pick], stream=st)
        batch.attend(0, qq, out, stream=st)
        outs.append((pick, qq, out))
        del batch
    torch.cuda.synchronize()
    for pick, qq, out in outs:
        assert right(out, codes, exps, table[pick], [kv_all[b] for b in pick], [1] * len(pick), qq)


@pytest.mark.parametrize("seqs,group,lens,q_max", [
    (4096, 1, (1, 90), 1), (1025, 2, (1, 200), 4), (200, 4, (1, 300), 12), (33, 8, (100, 700), 1)])
def test_many_sequences(seqs, group, lens, q_max):
    """More sequences than the plan's threads, some with nothing to do; the
    checked ones are a sample."""
    rng = np.random.default_rng(seqs)
    kv = rng.integers(*lens, seqs)
    ql = np.minimum(rng.integers(0, q_max + 1, seqs), kv)
    D, P, H, pages = 64, 64, 1, 600
    from ptxgen import KVCache
    codes, exps = ref.pool(rng, pages, H, P, D, spread=1.0)
    width = -(-int(kv.max()) // P)
    table = rng.integers(0, pages, (seqs, width)).astype(np.int32)     # pages shared for reading
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache = KVCache(pages, H, D, storage=(c, e))
    q = torch.from_numpy(rng.standard_normal((int(ql.sum()) + 2, H * group, D))).half().cuda()
    out = torch.full_like(q, 9.0)
    batch = cache.batch(table, kv, ql, stream=0)
    batch.attend(0, q, out, stream=0)
    batch.check_errors(stream=0)
    starts = np.r_[0, np.cumsum(ql)]
    got = out.cpu()
    assert (got[starts[-1]:] == 9.0).all()
    for b in rng.permutation(seqs)[:60]:
        rows = slice(starts[b], starts[b + 1])
        assert right(got[rows], codes, exps, table[b:b + 1], [int(kv[b])], [int(ql[b])], q[rows])


def test_addresses_past_32_bits():
    """A pool of 5 GB: pages at its end are appended to, copied and read."""
    from ptxgen import KVCache
    free, _ = torch.cuda.mem_get_info()
    if free < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    H, D, P, pages = 8, 128, 64, 40000
    cache = KVCache(pages, H, D)
    rng = np.random.default_rng(6)
    kv, first = [150], pages - 3
    table = np.array([[pages - 1, first, pages - 2]], np.int32)
    x = rng.standard_normal((2, 150, H, D)).astype(np.float16)
    k, v = (torch.from_numpy(a).cuda() for a in x)
    batch = cache.batch(table, kv, [150], stream=0)
    batch.append(0, k, v, stream=0)
    small = np.array([[2, 0, 1]], np.int32)
    codes, exps = ref.append(np.zeros((3, 2, H, P, D), np.uint8), np.zeros((3, 2, H), np.int8), small, kv, [150],
                             x[0].astype(float), x[1].astype(float))
    cache.copy_pages([pages - 1, first], [5, pages - 7], stream=0)
    moved = cache.batch([[5, pages - 7, pages - 2]], kv, [1], stream=0)
    for n, b in ((40, None), (1, moved), (150, batch)):
        b = b or cache.batch(table, kv, [n], stream=0)
        q = torch.from_numpy(rng.standard_normal((n, 2 * H, D))).half().cuda()
        out = torch.empty_like(q)
        b.attend(0, q, out, stream=0)
        torch.cuda.synchronize()
        assert right(out, codes, exps, small, kv, [n], q)
    cache.close()


def test_a_step_with_nothing_to_do():
    rng = np.random.default_rng(9)
    cache, codes, exps, table, q = make(rng, [70, 5], [1, 1])
    before = cache._storage[0].clone()
    batch = cache.batch(table, [70, 5], [0, 0], stream=0)
    out = torch.full_like(q, 3.0)
    batch.attend(0, q, out, stream=0)
    kv = torch.ones((2, 2, 128), device="cuda")
    batch.append(0, kv, kv, stream=0)
    batch.check_errors(stream=0)
    assert (out == 3.0).all() and (cache._storage[0] == before).all()


def test_a_plan_of_another_call_is_noticed():
    """attend with a plan made for other heads writes nothing."""
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(10)
    cache, codes, exps, table, q = make(rng, [70, 500], [1, 1])
    batch = cache.batch(table, [70, 500], stream=0)
    batch.reserve(8, stream=0)
    batch.reserve(4, stream=0)
    batch._plans[8, 0, 0] = batch._plans[4, 0, 0]
    out = torch.full_like(q, 3.0)
    batch.attend(0, q, out, stream=0)
    with pytest.raises(EmmyError, match="0x404"):
        batch.check_errors(stream=0)
    assert (out == 3.0).all()


def test_results_do_not_depend_on_the_cut():
    """One sequence alone, cut in many parts, and among many others, whole."""
    rng = np.random.default_rng(12)
    kv = [1800] + [600] * 400
    pages = 400
    from ptxgen import KVCache
    codes, exps = ref.pool(rng, pages, 2, 64, 64)
    c, e = torch.from_numpy(codes)[None].cuda(), torch.from_numpy(exps)[None].cuda()
    cache = KVCache(pages, 2, 64, storage=(c, e))
    table = rng.integers(0, pages, (401, 29)).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((401, 6, 64))).half().cuda()
    both = []
    for n in (1, 401):
        out = torch.empty_like(q[:n])
        cache.batch(table[:n], kv[:n], stream=0).attend(0, q[:n], out, stream=0)
        both.append(out[:1])
    for out in both:
        assert right(out, codes, exps, table[:1], kv[:1], [1], q[:1])


def test_more_new_tokens_than_max_q_are_reported():
    """Lengths that grew on the device past what the call was made for: the
    sequence is skipped, by either kernel and by append."""
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(13)
    for n in (1, 50):
        cache, codes, exps, table, q = make(rng, [200, 70], [n, 1])
        batch = cache.batch(table, [200, 70], [n, 1], stream=0)
        q = torch.cat([q, q])
        out = torch.full_like(q, 3.0)
        batch._d.tokens += 1                                 # q and out have more rows
        starts = np.array([0, n + 1, n + 2], np.int32)
        torch.cuda.synchronize()
        from ptxgen.kvcache import _copy_in
        _copy_in(cache.dev, batch._d.q_starts, starts, 0)
        batch.attend(0, q, out, stream=0)
        with pytest.raises(EmmyError, match="0x402"):
            batch.check_errors(stream=0)
        assert (out[:n + 1] == 3.0).all() and (out[n + 1] != 3.0).any() and (out[n + 2:] == 3.0).all()
        before = cache._storage[0].clone()
        k = torch.ones((2 * n + 2, 2, 128), device="cuda")
        batch.append(0, k, k, stream=0)
        with pytest.raises(EmmyError, match="0x402"):
            batch.check_errors(stream=0)
        changed = (before != cache._storage[0]).flatten(2).any(2)[0].nonzero().flatten().tolist()
        assert set(changed) <= {int(table[1, 1])}


def test_out_whose_rows_overlap_is_refused():
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(14)
    cache, codes, exps, table, q = make(rng, [70, 5, 9], [1, 1, 1])
    batch = cache.batch(table, [70, 5, 9], stream=0)
    one = torch.zeros((1, 8, 128), dtype=torch.float16, device="cuda")
    flat = torch.zeros(4096, dtype=torch.float16, device="cuda")
    for bad in (one.expand(3, 8, 128), flat.as_strided((3, 8, 128), (128, 128, 1)),
                flat.as_strided((3, 8, 128), (1024, 64, 1))):
        with pytest.raises(EmmyError, match="rows of out overlap"):
            batch.attend(0, q, bad, stream=0)
    heads_first = torch.zeros((8, 3, 128), dtype=torch.float16, device="cuda").transpose(0, 1)
    batch.attend(0, q, heads_first, stream=0)
    assert right(heads_first, codes, exps, table, [70, 5, 9], [1, 1, 1], q)
    with pytest.raises(EmmyError, match="q and out overlap"):
        batch.attend(0, q, q, stream=0)


def test_a_batch_used_on_another_stream_than_its_own():
    """No order given by the caller: the batch's lengths are there all the same."""
    rng = np.random.default_rng(15)
    cache, codes, exps, table, q = make(rng, [3000, 70], [1, 1])
    torch.cuda.synchronize()
    for _ in range(10):
        out = torch.zeros_like(q)
        batch = cache.batch(table, [3000, 70])               # the framework's stream
        batch.attend(0, q, out, stream=0)
        torch.cuda.synchronize()
        assert right(out, codes, exps, table, [3000, 70], [1, 1], q)


def test_q_of_extreme_rows():
    """Rows near the ends of bf16's range, zero rows, and rows with NaN."""
    rng = np.random.default_rng(16)
    kv, ql = [200, 65], [1, 40]
    cache, codes, exps, table, _ = make(rng, kv, ql, H=1, G=4, D=64, spread=0.0)
    q = rng.standard_normal((41, 4, 64))
    q[:, 0] *= 1e36
    q[:, 1] *= 1e-38
    q[:, 2] = 0
    q = torch.from_numpy(q).to(torch.bfloat16).cuda()
    q[:, 3, 5] = float("nan")
    out = torch.empty_like(q)
    cache.batch(table, kv, ql, stream=0).attend(0, q, out, scale=1e-3, stream=0)
    want, bound = ref.attend(codes, exps, table, kv, ql, q.float().cpu().numpy().astype(float), 1e-3)
    got = out.float().cpu().numpy()
    assert np.isnan(got[:, 3]).all()
    # scores of 1e34, whose own rounding decides which key takes all
    most = max(np.abs(x).max() for b in (0, 1) for x in ref.held(codes, exps, table, b, kv[b], 0)[1:])
    assert np.isfinite(got[:, 0]).all() and (np.abs(got[:, 0]) <= most * (1 + 2.0 ** -8)).all()
    assert (np.abs(got[:, 0]).max(1) > 0).all()
    assert ref.close(got[:, 1:3], want[:, 1:3], bound[:, 1:3], "bf16")


def test_what_a_capture_cannot_hold_is_refused():
    """Copies from the host, and the first attend of a batch, during a
    capture: refused, and the capture goes on."""
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(21)
    kv, ql = [300, 70], [1, 3]
    cache, codes, exps, table, q = make(rng, kv, ql)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    batch = cache.batch(table, kv, ql, stream=st)
    batch.reserve(q.shape[1], stream=st)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        for call in (lambda: cache.batch(table, kv, ql, stream=st), lambda: batch.update(table, kv, ql, stream=st),
                     lambda: batch.attend(0, q, out, window=64, stream=st), lambda: batch.check_errors(stream=st)):
            with pytest.raises(EmmyError, match="captured"):
                call()
        batch.attend(0, q, out, stream=st)
    graph.replay()
    torch.cuda.synchronize()
    assert right(out, codes, exps, table, kv, ql, q)


def test_a_scale_too_large_for_f32_is_refused():
    from ptxgen.runtime import EmmyError
    rng = np.random.default_rng(22)
    cache, codes, exps, table, q = make(rng, [70], [1])
    batch, out = cache.batch(table, [70], [1], stream=0), torch.empty_like(q)
    for scale in (3e38, -3e38, float("inf"), float("nan")):
        with pytest.raises(EmmyError, match="scale"):
            batch.attend(0, q, out, scale=scale, stream=0)


@pytest.mark.parametrize("D,window,sinks", [(64, 0, 0), (64, 100, 3), (128, 0, 0), (128, 200, 70)])
def test_many_units_of_one_and_two_tiles(D, window, sinks):
    """More units of the tile kernel than SMs, so that a CTA goes from one to
    the next: whole ones, ones with a single tile, histories of every length,
    and NaN values that only some of the units see."""
    rng = np.random.default_rng(23)
    H, G, B = 5, 2, 80
    ql = rng.integers(17, 300, B)
    ql[:6] = 128, 64, 65, 192, 256, 1
    kv = ql + np.where(rng.random(B) < 0.5, 0, rng.integers(0, 400, B))
    cache, codes, exps, table, q = make(rng, kv.tolist(), ql.tolist(), H=H, G=G, D=D)
    for b in (7, 20, 41):                           # one NaN each, in the middle of the keys
        at = int(kv[b]) // 2
        codes[table[b, at // 64], 1, b % H, at % 64, b] = 0x7f
    cache._storage[0].copy_(torch.from_numpy(codes)[None])
    batch, out = cache.batch(table, kv, ql, stream=0), torch.empty_like(q)
    torch.cuda.synchronize()
    for _ in range(2):
        batch.attend(0, q, out, window=window, sinks=sinks, stream=0)
    batch.check_errors(stream=0)
    assert right(out, codes, exps, table, kv, ql, q, window=window, sinks=sinks)
    first = out.clone()
    batch.attend(0, q, out, window=window, sinks=sinks, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("prompts,singles", [([700, 90], 40), ([33], 3), ([1500], 300)])
def test_prompts_beside_single_tokens_and_what_follows(prompts, singles):
    """Both kernels of a call run at once; what is queued after it (copies over
    every page it reads, at once, and a write to q) still comes after both."""
    rng = np.random.default_rng(24)
    ql = prompts + [1] * singles
    kv = [n + int(rng.integers(0, 300)) for n in prompts] + rng.integers(1, 1200, singles).tolist()
    used = sum(-(-n // 64) for n in kv)
    cache, codes, exps, table, q = make(rng, kv, ql, extra=used + 2)
    pages = sorted({int(table[b, i]) for b, n in enumerate(kv) for i in range(-(-n // 64))})
    spare = [p for p in range(cache.pages) if p not in set(pages)][:len(pages)]
    st = torch.cuda.current_stream()
    batch, out = cache.batch(table, kv, ql, stream=st), torch.empty_like(q)
    batch.attend(0, q, out, stream=st)
    batch.check_errors(stream=st)
    assert right(out, codes, exps, table, kv, ql, q)
    want, kept, q0 = out.clone(), [x.clone() for x in cache._storage], q.clone()
    for _ in range(10):
        for x, y in zip(cache._storage, kept):
            x.copy_(y)
        q.copy_(q0)
        out.zero_()
        batch.attend(0, q, out, stream=st)
        cache.copy_pages(spare[:len(pages)], pages, stream=st)
        q.zero_()
        assert torch.equal(out, want)
    batch.check_errors(stream=st)
