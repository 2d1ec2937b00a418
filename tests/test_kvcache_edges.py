"""The cache's host side where calls meet: collections inside its own locks."""

import threading

from ptxgen import kvcache as kv
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
