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


def write(cache, s, slots, tokens):
    """What a step does with the slots: the pages they lie in have to be this sequence's alone."""
    size = cache.page_tokens
    for slot, token in zip(slots, tokens):
        assert slot // size in s.pages and cache.holders(slot // size) == 1
        cache.memory[slot] = token


def read(cache, s):
    size = cache.page_tokens
    apply_copies(cache)
    return [cache.memory[s.pages[t // size] * size + t % size] for t in range(s.tokens)]


def apply_copies(cache):
    size = cache.page_tokens
    for (a, b), rows, _ in cache.context.copied:
        for r in range(size):
            cache.memory.pop(b * size + r, None)
        cache.memory.update({b * size + r: cache.memory[a * size + r] for r in range(rows)})
    cache.context.copied.clear()


@pytest.mark.parametrize("cut,more", [(20, 4), (17, 1), (31, 1), (31, 20), (5, 40), (32, 3), (16, 3)])
def test_a_fork_that_is_cut_back_writes_to_pages_of_its_own(cache, cut, more):
    cache.memory = {}
    a = cache.sequence()
    write(cache, a, a.extend(40), range(40))
    b = a.fork(stream=3)
    for s, name in ((a, 1000), (b, 2000)):  # the one that is cut first, then the other
        s.truncate(cut)
        slots = s.extend(more, stream=3)
        apply_copies(cache)
        write(cache, s, slots, range(name, name + more))
        if s is a:
            assert read(cache, b) == list(range(40))
    assert read(cache, a) == [*range(cut), *range(1000, 1000 + more)] and read(cache, b) == [*range(cut), *range(2000, 2000 + more)]
    for s in (a, b):
        s.free()
    assert cache.free_pages() == 60


def test_the_last_holder_writes_in_place(cache):
    a = cache.sequence()
    a.extend(32)
    b = a.fork()
    a.truncate(20)
    b.free()
    page = a.pages[1]
    assert a.extend(0) == [] and a.extend(2) == [page * 16 + 4, page * 16 + 5] and not cache.context.copied


def test_an_extension_that_cannot_be_changes_nothing(cache):
    a = cache.sequence()
    a.extend(32)
    b = a.fork()
    a.truncate(20)
    rest = cache.sequence()
    rest.extend(16 * (cache.free_pages() - 1))
    pages = list(a.pages)
    with pytest.raises(N.WfError):
        a.extend(13)  # a copy of the shared page and one more
    assert a.pages == pages and a.tokens == 20 and cache.free_pages() == 1 and cache.holders(pages[1]) == 2
    for fail in ("allocate", "copy", "copy_pages"):
        cache.context.fail = (fail,)
        with pytest.raises(MemoryError):
            a.extend(12)
        assert a.pages == pages and a.tokens == 20 and cache.free_pages() == 1 and cache.holders(pages[1]) == 2
    cache.context.fail = ()
    a.extend(12)
    assert cache.free_pages() == 0 and a.pages[0] == b.pages[0] and a.pages[1] != b.pages[1]


def test_sequences_against_lists(cache):
    """Growing, cutting and forking at random: every sequence reads what was written to it."""
    rng, cache.memory, live, number = random.Random(5), {}, [], 0
    for _ in range(3000):
        what = rng.random()
        if not live or what < 0.05:
            live.append((cache.sequence(), []))
            continue
        s, text = rng.choice(live)
        try:
            if what < 0.5:
                n = rng.choice((0, 1, 1, 5, 16, 37))
                slots = s.extend(n)
                apply_copies(cache)
                new = list(range(number, number + n))
                number += n
                write(cache, s, slots, new)
                text += new
            elif what < 0.7:
                n = rng.randint(0, s.tokens)
                s.truncate(n)
                del text[n:]
            elif what < 0.85:
                live.append((s.fork(), list(text)))
            else:
                s.free()
                live = [x for x in live if x[0] is not s]
        except N.WfError as e:
            assert e.status == N.WF_ERR_TOO_LARGE
            live[0][0].free()
            del live[0]
        for t, want in live:
            assert read(cache, t) == want
        held = [p for t, _ in live for p in t.pages]
        assert cache.free_pages() == 60 - len(set(held)) and all(cache.holders(p) == held.count(p) for p in set(held))


def test_pages_are_made_private_before_tokens_move(cache):
    a = cache.sequence()
    a.extend(50)
    b, c = cache.fork([a, a])
    before = list(b.pages)
    cache.context.copied.clear()
    cache.own([a, b], [(20, 22), (33, 33)], stream=5)
    assert cache.context.copied == [((before[1], a.pages[1]), 16, 5)]
    assert a.pages[0] == b.pages[0] and a.pages[1] not in (before[1],) and a.pages[2] == before[2] and b.pages == before
    cache.context.copied.clear()
    cache.own([b, c], [(0, 48), (15, 33)])  # page 1 has two holders left: one copy is enough
    moved = [pair for pair, _, _ in cache.context.copied]
    assert len(moved) == 3 + 3 - 1 and not set(b.pages) & set(c.pages[:3])
    for s in (a, b, c):
        s.free()
    assert cache.free_pages() == 60


@pytest.mark.parametrize("fail", ["allocate", "second allocate", "pool"])
def test_a_cache_that_cannot_be_made_holds_no_memory(fail):
    from warpforge_b200.attention import KvCache

    ctx = Context()
    ctx.fail = (fail,)
    if fail == "pool":
        ctx._lib.wf_pages_create = lambda pages, pool: N.WF_ERR_SHAPE
    with pytest.raises((MemoryError, N.WfError)):
        KvCache(ctx, layers=2, pages=60, page_tokens=16, kv_heads=1, head_dim=64)
    assert not ctx.live
