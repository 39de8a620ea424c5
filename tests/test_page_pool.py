"""The page pool behind KvCache (wf_pages_*): host bookkeeping, no device."""
import ctypes
import random

import pytest

from warpforge_b200 import _native as N

LIB = N.load()


@pytest.fixture
def pool():
    h = ctypes.c_int64()
    assert LIB.wf_pages_create(10, ctypes.byref(h)) == N.WF_OK
    yield h.value
    LIB.wf_pages_destroy(h.value)


def take(pool, n):
    ids = (ctypes.c_int32 * max(n, 1))()
    rc = LIB.wf_pages_take(pool, n, ids)
    return rc, list(ids)[:n]


def ids(*v):
    return (ctypes.c_int32 * len(v))(*v)


def free(pool):
    total, left = ctypes.c_int64(), ctypes.c_int64()
    assert LIB.wf_pages_info(pool, ctypes.byref(total), ctypes.byref(left)) == N.WF_OK and total.value == 10
    return left.value


def holders(pool, i):
    n = ctypes.c_int64()
    assert LIB.wf_pages_holders(pool, i, ctypes.byref(n)) == N.WF_OK
    return n.value


def test_lowest_pages_first_all_or_none(pool):
    assert take(pool, 3) == (N.WF_OK, [0, 1, 2])
    assert take(pool, 8)[0] == N.WF_ERR_TOO_LARGE and free(pool) == 7
    assert LIB.wf_pages_release(pool, 1, ids(1)) == N.WF_OK
    assert take(pool, 2) == (N.WF_OK, [1, 3])
    assert take(pool, 0) == (N.WF_OK, [])


def test_shared_pages_end_with_their_last_holder(pool):
    take(pool, 2)
    assert LIB.wf_pages_share(pool, 2, ids(0, 0)) == N.WF_OK and holders(pool, 0) == 3 and holders(pool, 5) == 0
    assert LIB.wf_pages_release(pool, 3, ids(0, 1, 0)) == N.WF_OK
    assert holders(pool, 0) == 1 and holders(pool, 1) == 0 and free(pool) == 9
    assert LIB.wf_pages_release(pool, 1, ids(0)) == N.WF_OK and free(pool) == 10
    assert take(pool, 10) == (N.WF_OK, list(range(10)))


def test_refusals_change_nothing(pool):
    take(pool, 3)
    assert LIB.wf_pages_release(pool, 3, ids(0, 1, 1)) == N.WF_ERR_INDEX  # named more often than held
    assert LIB.wf_pages_release(pool, 2, ids(2, 9)) == N.WF_ERR_INDEX
    assert LIB.wf_pages_release(pool, 1, ids(-1)) == N.WF_ERR_INDEX
    assert LIB.wf_pages_share(pool, 2, ids(0, 7)) == N.WF_ERR_INDEX
    assert [holders(pool, i) for i in range(4)] == [1, 1, 1, 0] and free(pool) == 7
    assert LIB.wf_pages_take(pool, -1, ids(0)) == N.WF_ERR_INVALID_ARGUMENT
    assert LIB.wf_pages_take(pool, 1, None) == N.WF_ERR_INVALID_ARGUMENT
    n = ctypes.c_int64()
    assert LIB.wf_pages_holders(pool, 10, ctypes.byref(n)) == N.WF_ERR_INDEX
    assert LIB.wf_pages_create(-1, ctypes.byref(n)) == N.WF_ERR_SHAPE
    assert LIB.wf_pages_create(1, None) == N.WF_ERR_INVALID_ARGUMENT
    for call in (lambda: LIB.wf_pages_destroy(0), lambda: LIB.wf_pages_destroy(12345), lambda: take(77, 1)[0], lambda: LIB.wf_pages_info(77, None, None)):
        assert call() == N.WF_ERR_INVALID_HANDLE


def test_against_counts(pool):
    rng = random.Random(3)
    held = [0] * 10
    for _ in range(2000):
        live = [i for i, n in enumerate(held) if n]
        what = rng.random()
        if what < 0.4:
            n = rng.randint(0, 4)
            rc, got = take(pool, n)
            spare = [i for i, c in enumerate(held) if not c]
            if n > len(spare):
                assert rc == N.WF_ERR_TOO_LARGE
                continue
            assert rc == N.WF_OK and got == spare[:n]
            for i in got:
                held[i] = 1
        elif live:
            pick = [rng.choice(live) for _ in range(rng.randint(1, 4))]
            if what < 0.6:
                assert LIB.wf_pages_share(pool, len(pick), ids(*pick)) == N.WF_OK
                for i in pick:
                    held[i] += 1
            else:
                fits = all(pick.count(i) <= held[i] for i in pick)
                assert LIB.wf_pages_release(pool, len(pick), ids(*pick)) == (N.WF_OK if fits else N.WF_ERR_INDEX)
                if fits:
                    for i in pick:
                        held[i] -= 1
        assert [holders(pool, i) for i in range(10)] == held and free(pool) == held.count(0)


def test_calls_without_a_context():
    args, cache = N.TreeAttentionArgs(), N.KvCacheArgs()
    for fn, a in ((LIB.wf_tree_attention, args), (LIB.wf_prompt_attention, N.PromptAttentionArgs()), (LIB.wf_qk_norm_rope, N.QkNormRopeArgs())):
        assert fn(77, ctypes.byref(a), ctypes.byref(cache), 0, 0) == N.WF_ERR_INVALID_HANDLE
    assert LIB.wf_cache_copy_pages(77, ctypes.byref(cache), 0, 0, 0, 0) == N.WF_ERR_INVALID_HANDLE
    assert LIB.wf_cache_compact(77, ctypes.byref(cache), 0, 0, 0, 0, 0, 0, 0, 0) == N.WF_ERR_INVALID_HANDLE


def test_structs_are_laid_out_as_the_header_says():
    assert [ctypes.sizeof(t) for t in (N.KvCacheArgs, N.QkNormRopeArgs, N.PromptAttentionArgs, N.TreeAttentionArgs)] == [40, 136, 80, 96]


def test_rope_table():
    import numpy as np

    from warpforge_b200.attention import rope_table

    t = rope_table(5, 8, 100.0, factors=np.array([1, 1, 2, 2]))
    assert t.shape == (5, 4, 2) and t.dtype == np.float32
    assert np.allclose(t[3, 1], [np.cos(3 * 100 ** -0.25), np.sin(3 * 100 ** -0.25)]) and np.allclose(t[3, 2, 0], np.cos(3 * 100 ** -0.5 / 2))
    with pytest.raises(ValueError):
        rope_table(5, 7)


class HostContext:
    """A context without a device: addresses are numbers, copies are kept, kernels are not launched."""

    def __init__(self, lib):
        self._lib, self.handle, self.freed, self.copies = lib, 0, [], []
        self._next = 4096

    def _ck(self, what, status):
        pass

    def allocate(self, n):
        self._next += -(-n // 256) * 256
        return self._next

    def free(self, p):
        self.freed.append(p)

    def copy_to_device(self, dptr, host, stream=0, sync=True):
        self.copies.append((dptr, host.tolist(), stream))


@pytest.fixture
def cache():
    from warpforge_b200.attention import KvCache

    made = KvCache(HostContext(LIB), layers=2, pages=12, page_tokens=16, kv_heads=1, head_dim=64)
    yield made
    made.close()


def test_forks_of_two_streams_have_arrays_of_their_own(cache):
    a = cache.sequence()
    a.extend(20)
    forks = [a.fork(stream) for stream in (7, 8, 7)]
    assert [f.pages[0] for f in forks] == [a.pages[0]] * 3 and cache.holders(a.pages[0]) == 4
    at = {stream: {p for p, _, s in cache.context.copies if s == stream} for stream in (7, 8)}
    assert len(at[7]) == len(at[8]) == 2 and not at[7] & at[8]
    pairs = [x for _, x, _ in cache.context.copies[::2]]
    assert pairs == [[[a.pages[1], f.pages[1]]] for f in forks]


def test_a_fork_that_cannot_be_changes_nothing(cache):
    a, b = cache.sequence(), cache.sequence()
    a.extend(20)
    b.extend(20)
    gone = list(b.pages)
    cache._release(gone)  # b names pages that nobody holds
    free = cache.free_pages()
    with pytest.raises(Exception):
        cache.fork([a, b])
    assert cache.free_pages() == free and [cache.holders(p) for p in a.pages] == [1, 1]
    b.pages, b.tokens = [], 0
    c = cache.sequence()
    c.extend(16 * cache.free_pages())  # no page is left for the part-full one
    with pytest.raises(Exception):
        a.fork()
    assert cache.free_pages() == 0 and [cache.holders(p) for p in a.pages] == [1, 1]


def test_a_sequence_forked_twice_in_one_call(cache):
    a = cache.sequence()
    a.extend(33)
    one, two = cache.fork([a, a])
    assert cache.holders(a.pages[0]) == cache.holders(a.pages[1]) == 3
    assert len({a.pages[2], one.pages[2], two.pages[2]}) == 3
    for s in (a, one, two):
        s.free()
    assert cache.free_pages() == 12
