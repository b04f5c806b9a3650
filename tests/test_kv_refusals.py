"""More of what the kv entry points refuse, on the host: a pool that was freed,
rotation bases without angles."""
import pytest

import rce_amd
from test_kv_args import BAD, NULL, append, attend, batch, cache, read, refused


class Buffer:
    freed = False

    def free(self):
        self.freed = True


@pytest.mark.parametrize("call", [append, read, attend])
def test_a_freed_pool(call):
    c = cache()
    c.buffers = own = tuple(Buffer() for _ in range(4))  # as KvCache.allocate leaves it
    sizes = c.sizes()
    c.free()
    assert all(b.freed for b in own) and c.sizes() == sizes
    refused(NULL, call, c, batch())
    c.free()


def test_the_callers_own_pool_stays_its_own():
    c = cache()
    raw = c.raw
    c.free()
    assert c.raw == raw


def test_rotation_bases_without_angles():
    for base in (float("inf"), float("nan"), 0.0, -1.0):
        refused(BAD, rce_amd.Rope.table, base, 8, 5)
