"""Sequences of a KvCache that share pages: what they hold, and what happens where something fails.  Host bookkeeping, no device."""
import ctypes
import random

import pytest

from warpforge_b200 import _native as N

LIB = N.load()


class Library:
    """The native library; calls that would launch a kernel are noted instead."""

    def __init__(self, context):
        self._context = context

    def __getattr__(self, name):
        return getattr(LIB, name)

    def wf_cache_copy_pages(self, handle, cache, pairs, rows, n, stream):
        c = self._context
        c.step("copy_pages")
        at = {p: v for p, v, s in c.copies if s == stream}  # the last copy to each address
        assert len(at[pairs]) == len(at[rows]) == n
        c.copied += [(tuple(pair), r, stream) for pair, r in zip(at[pairs], at[rows])]
        return N.WF_OK


class Context:
    """A context without a device.  fail: the names of the calls that raise."""

    def __init__(self):
        self._lib, self.handle, self.live, self.copies, self.copied, self.fail = Library(self), 1, {}, [], [], ()
        self._next = 4096

    def _ck(self, what, status):
        N.check(what, status)

    def step(self, name):
        if name in self.fail:
            raise MemoryError(name)

    def allocate(self, n):
        self.step("allocate")
        if "second allocate" in self.fail:
            self.fail = ("allocate",)
        self._next += -(-n // 256) * 256
        self.live[self._next] = n
        return self._next

    def free(self, p):
        del self.live[p]

    def copy_to_device(self, dptr, host, stream=0, sync=True):
        self.step("copy")
        assert host.nbytes <= self.live[dptr]
        self.copies.append((dptr, host.tolist(), stream))


@pytest.fixture
def cache():
    from warpforge_b200.attention import KvCache

    made = KvCache(Context(), layers=2, pages=60, page_tokens=16, kv_heads=1, head_dim=64)
    yield made
    made.context.fail = ()
    made.close()
    assert not made.context.live


@pytest.mark.parametrize("fail", ["allocate", "second allocate"])
def test_arrays_of_forks_that_cannot_grow(cache, fail):
    """Where larger arrays cannot be had the old ones are still there, and each is freed once."""
    a = cache.sequence()
    a.extend(5)
    few = a.fork()
    before = dict(cache.context.live)
    cache.context.fail = (fail,)
    with pytest.raises(MemoryError):
        cache.fork([a] * 20)
    assert cache.context.live == before
    again = a.fork()
    assert cache.context.copied[-1] == ((a.pages[0], again.pages[0]), 5, 0)
    cache.context.fail = ()
    assert len({s.pages[0] for s in cache.fork([a] * 20) + [few, again]}) == 22


@pytest.mark.parametrize("fail", ["allocate", "second allocate", "copy", "copy_pages"])
def test_a_fork_that_fails_late_holds_nothing(cache, fail):
    a, b = cache.sequence(), cache.sequence()
    a.extend(40)
    b.extend(33)
    free, holders = cache.free_pages(), [cache.holders(p) for p in a.pages + b.pages]
    cache.context.fail = (fail,)
    with pytest.raises(MemoryError):
        cache.fork([a, b, a])
    assert cache.free_pages() == free and [cache.holders(p) for p in a.pages + b.pages] == holders
    cache.context.fail = ()
    c = a.fork()
    for s in (a, b, c):
        s.free()
    assert cache.free_pages() == 60
