"""Bounded waits of the cache's attention kernels that run out: all, half or a
third of the blocks wait for an arrival that they withhold themselves, with the
limit at a millisecond.  The kernels report it and end, and the same batch then
computes as if nothing had been (no fault, no endless loop: a block whose wait
has run out lets its copies land and goes on to its end)."""

import numpy as np
import pytest

from tests import kv8_oracle as ref
from tests.test_gpu_kvcache import NP, cache_of, gpu  # noqa: F401 - a fixture

pytestmark = pytest.mark.gpu


# one segment as a cluster; some in clusters of four; single parts; units that
# were cut; both kernels
@pytest.mark.parametrize("H,G,D,seqs", [
    (1, 4, 128, [(400, 1)]),
    (2, 8, 64, [(30000, 1)]),
    (2, 2, 128, [(9000, 1)] + [(300 + i, 1) for i in range(40)]),
    (1, 4, 128, [(3000, 40)]),
    (2, 4, 64, [(700, 300), (900, 1), (3000, 2)]),
])
def test_waits_that_run_out(gpu, H, G, D, seqs):  # noqa: F811
    from ptxgen.kvcache import WORKSPACE_ZERO
    from ptxgen.runtime import EmmyError, load_library
    rng = np.random.default_rng(3)
    P = 64
    kv, ql = [a for a, _ in seqs], [b for _, b in seqs]
    pages = sum(-(-n // P) for n in kv)
    codes, exps = ref.pool(rng, pages, H, P, D)
    table = ref.tables(rng, pages, kv, P)
    q = rng.standard_normal((sum(ql), H * G, D)).astype(NP["f16"])
    cache, _, _ = cache_of(gpu, codes[None], exps[None])
    batch = cache.batch(table, kv, ql)
    qd, od = gpu.put(q, "f16"), gpu.put(np.zeros_like(q), "f16")
    L = load_library()
    want, bound = ref.attend(codes, exps, table, kv, ql, q.astype(float), D ** -0.5)
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
        assert ref.close(gpu.get(od, q.shape, np.float16), want, bound, "f16")
    batch.close()
