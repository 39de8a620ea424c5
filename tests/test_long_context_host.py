"""Shared prefixes, bounds and lists as far as they need no device: which prefixes a cache finds, refusals of shapes and types, a decoder's buffers."""
import itertools

import numpy as np
import pytest

from test_generate_host import HostContext as ClosedContext

from warpforge_b200 import attention as A
from warpforge_b200.backend import DeviceTensor


class HostContext(ClosedContext):
    """... that counts as open: what is closed gives its memory back."""

    def __init__(self):
        super().__init__()
        self.handle = 0x1234


def dev(dtype, *shape, ptr=4096):
    return DeviceTensor(ptr, shape, dtype)


@pytest.fixture
def cache():
    c = A.KvCache(HostContext(), 2, 64, 16, 2, 64)
    yield c
    c.close()


def made(cache, pages, tokens):
    return A.Sequence(cache, pages, tokens)


def pages_read(groups, prefix, tokens, size):
    """Whole pages that a call reads: a prefix once a group, the rest of every sequence."""
    read = 0
    for g, p in enumerate(prefix):
        members = range(groups[g], groups[g + 1])
        read += p // size + sum(tokens[s] // size - p // size for s in members)
    return read


def check_groups(cache, sequences, tokens=None):
    groups, prefix = cache.shared_prefixes(sequences, tokens)
    lens = [s.tokens for s in sequences] if tokens is None else tokens
    assert groups.dtype == prefix.dtype == np.int32 and groups[0] == 0 and groups[-1] == len(sequences) and len(groups) == len(prefix) + 1
    for g, p in enumerate(prefix):
        members = sequences[groups[g]:groups[g + 1]]
        assert len(members) >= 1 and p % 16 == 0 and (p == 0 or len(members) > 1)
        assert len({tuple(s.pages[:p // 16]) for s in members}) == 1
        assert all(p <= n for n in lens[groups[g]:groups[g + 1]])
    return groups, prefix


def test_prefixes_of_forks(cache):
    seqs = [made(cache, [1, 2, 3, 4], 60), made(cache, [1, 2, 3, 9], 50), made(cache, [1, 2, 3, 7, 8], 75)]
    assert [x.tolist() for x in check_groups(cache, seqs)] == [[0, 3], [48]]
    assert [x.tolist() for x in check_groups(cache, seqs, [47, 50, 75])] == [[0, 3], [32]]
    assert [x.tolist() for x in check_groups(cache, seqs + [made(cache, [20, 2], 32)])] == [[0, 3, 4], [48, 0]]
    assert [x.tolist() for x in check_groups(cache, [made(cache, [5], 9), made(cache, [5], 9)])] == [[0, 1, 2], [0, 0]]  # no whole page
    assert [x.tolist() for x in check_groups(cache, [seqs[0]])] == [[0, 1], [0]]
    assert [x.tolist() for x in check_groups(cache, [made(cache, [], 0), made(cache, [], 0)])] == [[0, 1, 2], [0, 0]]
    assert check_groups(cache, [])[0].tolist() == [0]


def test_prefixes_leave_the_fewest_pages(cache):
    """Against all ways to cut the line."""
    rng = np.random.default_rng(0)
    for _ in range(60):
        n = int(rng.integers(1, 8))
        seqs = [made(cache, list(range(100, 100 + int(rng.integers(0, 5)))) + list(range(200 + 10 * i, 203 + 10 * i)), 0) for i in range(n)]
        for s in seqs:
            s.tokens = 16 * len(s.pages) - int(rng.integers(0, 20))
        tokens = [s.tokens for s in seqs]
        groups, prefix = check_groups(cache, seqs)
        best = None
        for cuts in itertools.product((0, 1), repeat=n - 1):
            at = [0] + [i + 1 for i, c in enumerate(cuts) if c] + [n]
            pre = []
            for a, b in zip(at, at[1:]):
                m = min(t // 16 for t in tokens[a:b])
                while len({tuple(s.pages[:m]) for s in seqs[a:b]}) > 1:
                    m -= 1
                pre.append(16 * m if b - a > 1 else 0)
            read = pages_read(at, pre, tokens, 16)
            best = read if best is None else min(best, read)
        assert pages_read(groups, prefix, tokens, 16) == best


def test_bounds_refuse(cache):
    with pytest.raises(ValueError):
        A.PageBounds(cache, codes=dev("i8", 2, 64, 2, 2, 64))
    with pytest.raises(ValueError):
        A.PageBounds(cache, codes=dev("i8", 2, 64, 2, 64), scales=dev("f32", 2, 64, 2))
    with pytest.raises(ValueError):
        A.PageBounds(cache, codes=dev("bf16", 2, 64, 2, 2, 64), scales=dev("f32", 2, 64, 2))
    b = A.PageBounds(cache, codes=dev("i8", 2, 64, 2, 2, 64), scales=dev("f32", 2, 64, 2, ptr=1 << 20))
    codes, scales = b.layer(1)
    assert (codes.ptr, codes.shape(), codes.nbytes()) == (4096 + 64 * 2 * 2 * 64, (64, 2, 2, 64), 64 * 2 * 2 * 64)
    assert (scales.ptr, scales.shape()) == ((1 << 20) + 64 * 2 * 4, (64, 2))
    for i in (-1, 2):
        with pytest.raises(ValueError):
            b.layer(i)
    with pytest.raises(ValueError):
        b.update(dev("i32", 3, 4), dev("i32", 3), dev("i32", 2), max_tokens=1)
    with pytest.raises(ValueError):
        b.update(dev("i64", 3, 4), dev("i32", 3), dev("i32", 3), max_tokens=1)


def test_bounds_that_cannot_be_made_give_their_memory_back():
    class Short(HostContext):
        def allocate(self, n):
            if n == 2 * 64 * 2 * 4:
                raise MemoryError
            return super().allocate(n)

    ctx = Short()
    c = A.KvCache(ctx, 2, 64, 16, 2, 64)
    held = len(ctx.room)
    with pytest.raises(MemoryError):
        A.PageBounds(c)
    assert len(ctx.room) == held
    c.close()


def test_operators_refuse():
    ctx = HostContext()
    q, kv, table, n = dev("bf16", 3, 4, 64), dev("bf16", 9, 2, 16, 64), dev("i32", 3, 5), dev("i32", 3)
    codes, scales, lists, lens = dev("i8", 9, 2, 2, 64), dev("f32", 9, 2), dev("i32", 3, 2, 6), dev("i32", 3, 2, 2)

    def select(q=q, codes=codes, scales=scales, lists=lists, lens=lens, **more):
        return A.SelectPages(ctx, q, codes, scales, table, n, lists, lens, page_tokens=16, max_context=50, **more)

    select()
    for bad in (dict(codes=dev("i8", 9, 2, 2, 32)), dict(scales=dev("f32", 9, 1)), dict(lists=dev("i32", 3, 4, 6)), dict(lens=dev("i32", 3, 2)), dict(q=dev("f32", 3, 4, 64)),
                dict(q_offsets=dev("i32", 3))):
        with pytest.raises(ValueError):
            select(**bad)

    def selected(q=q, lists=lists, lens=lens, out=q, **more):
        return A.SelectedAttention(ctx, q, kv, kv, out, lists, lens, **more)

    selected()
    for bad in (dict(lists=dev("i32", 3, 1, 6)), dict(lens=dev("i64", 3, 2, 2)), dict(out=dev("bf16", 3, 4, 32)), dict(ancestors=dev("i64", 2)), dict(q=dev("bf16", 2, 4, 64))):
        with pytest.raises(ValueError):
            selected(**bad)

    def shared(groups=dev("i32", 3), prefix=dev("i32", 2), **more):
        return A.SharedPrefixAttention(ctx, q, kv, kv, q, table, n, groups, prefix, max_prefix=16, max_own=16, **more)

    shared()
    for bad in (dict(groups=dev("i32", 2)), dict(prefix=dev("i64", 2)), dict(ancestors=dev("i64", 4)), dict(q_offsets=dev("i32", 5))):
        with pytest.raises(ValueError):
            shared(**bad)


def decoder(**more):
    from warpforge_b200.generate import Decoder, DecoderSpec
    from warpforge_b200.quant import QuantizationType

    return Decoder(HostContext(), DecoderSpec(QuantizationType.Q8_0, 64, 2, 1, 32, 64, 2, 64, max_positions=200), pages=30, page_tokens=16, max_tokens=32, max_sequences=3, **more)


def test_decoder_refuses():
    for bad in (dict(selected_pages=-1), dict(selected_pages=9, share_prefixes=True), dict(selected_pages=9, recent_tokens=-1), dict(selected_pages=2, recent_tokens=16),
                dict(selected_pages=9, first_pages=-1)):
        with pytest.raises(ValueError):
            decoder(**bad)
    m = decoder(selected_pages=4, first_pages=1, recent_tokens=16)
    s = m.sequence()
    m.prefill([s], [np.arange(20)])
    with pytest.raises(ValueError):
        m.step([s], [list(range(18))])  # 1 + (16 + 18 + 14) / 16 + 1 = 5
    assert s.tokens == 20
    m.step([s], [list(range(17))])
    m.close()
    assert not m.ctx.room


@pytest.mark.parametrize("more", [dict(share_prefixes=True), dict(selected_pages=12, recent_tokens=0)])
def test_decoder_runs_its_path(more):
    """Calls, copies and buffers of steps, forks and kept drafts, without a device."""
    m = decoder(**more)
    a = m.sequence()
    m.prefill([a], [np.arange(32) % 64])
    b = a.fork()
    m.prefill([a, b], [np.arange(3), np.arange(0)])
    m.step([a, b], [[1], [2]])
    m.step([a, b], [[1, 2, 3], [4]], [[-1, -1, 0], [-1]])
    m.keep([a, b], [3, 1], [[0, 2], []])
    assert (a.tokens, b.tokens) == (38, 33)
    m.step([a, b], [[], [3]])
    if m.share_prefixes:
        assert [x.tolist() for x in m.cache.shared_prefixes([a, b])] == [[0, 2], [32]]
    for s in (a, b):
        s.free()
    assert m.cache.free_pages() == 30
    m.close()
    assert not m.ctx.room
