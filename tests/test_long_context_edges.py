"""A decoder that selects pages or shares prefixes, as far as it needs no device: which bounds it asks for, which memory it holds, what its command takes."""
import numpy as np
import pytest

from test_long_context_host import HostContext, dev

from warpforge_b200 import attention as A
from warpforge_b200 import generate
from warpforge_b200.backend import DeviceTensor
from warpforge_b200.generate import Decoder, DecoderSpec
from warpforge_b200.quant import QuantizationType


class Watched(HostContext):
    """... that knows what was copied where."""

    def __init__(self):
        super().__init__()
        self.sent = {}

    def copy_to_device(self, dptr, host, stream=0, sync=True):
        super().copy_to_device(dptr, host, stream, sync)
        self.sent[dptr] = host.copy()


def decoder(max_tokens=64, max_sequences=4, **more):
    spec = DecoderSpec(QuantizationType.Q8_0, 64, 2, 1, 32, 64, 1, 64, max_positions=200)
    return Decoder(Watched(), spec, pages=30, page_tokens=16, max_tokens=max_tokens, max_sequences=max_sequences, selected_pages=12, recent_tokens=0, **more)


def watch_bounds(m):
    """Pages and rows of every update that follows."""
    seen = []

    def update(tables, first, stop, *, max_tokens):
        table, first, stop = (m.ctx.sent[x.ptr].reshape(x.shape()) for x in (tables, first, stop))
        now = []
        for row, a, b in zip(table, first, stop):
            assert 0 <= a <= b and b - a <= max_tokens
            now += [(int(row[j]), min(16, int(b) - 16 * j)) for j in range(a // 16, -(-b // 16))] if a < b else []
        assert len({page for page, _ in now}) == len(now), "a page by two sequences"
        for page, rows in now:
            assert rows == 16 or m.cache.holders(page) == 1, f"{rows} rows of page {page}, which others hold too"
        seen.append(now)

    m.bounds.update = update
    return seen


def test_kept_drafts_leave_the_bounds_of_pages_that_others_hold():
    """A fork between step and keep holds a page whole of which keep retains a part, at its place."""
    m = decoder()
    a = m.sequence()
    m.prefill([a], [np.arange(10)])
    seen = watch_bounds(m)
    m.step([a], [[0] * 6])
    assert seen == [[(a.pages[0], 16)]]
    b = a.fork()
    m.keep([a], [6], [[0, 1]])
    assert a.pages == b.pages and (a.tokens, b.tokens) == (12, 16) and [x for now in seen[1:] for x in now] == []
    m.step([a, b], [[0], [0]])
    assert a.pages[0] != b.pages[0] and seen[-1] == [(a.pages[0], 13), (b.pages[1], 1)]
    m.keep([a, b], [1, 1], [[0], [0]])
    # both branches in one call: one keeps what lies at its place, the other one moves tokens
    c = m.sequence()
    m.prefill([c], [np.arange(10)])
    m.step([c], [[0] * 22], [[-1] * 22])
    d, e = c.fork(), c.fork()
    m.keep([c, d, e], [22] * 3, [[0, 1], list(range(22)), [0, 3, 4]])
    assert c.pages[0] == d.pages[0] != e.pages[0] and seen[-1] == [(e.pages[0], 13)]
    m.step([c, d, e], [[0]] * 3)
    for s in (a, b, c, d, e):
        s.free()
    assert m.cache.free_pages() == 30
    m.close()


def test_full_pages_have_bounds_of_all_their_rows():
    """Steps, forks and keeps at random: what the last update of a page says is what a sequence that holds it full has."""
    rng = np.random.default_rng(5)
    for _ in range(30):
        m = decoder()
        seqs, rows = [m.sequence()], {}
        seen = watch_bounds(m)
        m.prefill(seqs, [np.arange(int(rng.integers(1, 50)))])
        for _ in range(12):
            n = [int(rng.integers(0, 12)) for _ in seqs]
            m.step(seqs, [[0] * k for k in n], [[-1] * k for k in n])
            if len(seqs) < 4 and rng.random() < 0.5:
                i = int(rng.integers(len(seqs)))
                seqs.append(seqs[i].fork())
                n.append(n[i])
            kept = [sorted(rng.choice(k, int(rng.integers(0, k + 1)), replace=False).tolist()) if rng.random() < 0.5 else list(range(int(rng.integers(0, k + 1)))) for k in n]
            m.keep(seqs, n, kept)
            for now in seen:
                rows.update(now)
            seen.clear()
            for s in seqs:
                for page in s.pages[:s.tokens // 16]:
                    assert rows[page] == 16
                if s.tokens > 100:
                    s.truncate(int(rng.integers(1, 40)))
        for s in seqs:
            s.free()
        m.close()


def test_lists_have_room_for_the_tokens_of_a_step():
    """... which are no more than 64 for each sequence, however long prompts are."""
    for max_tokens, max_sequences, tokens in ((4096, 2, 128), (50, 2, 50), (128, 2, 128)):
        m = decoder(max_tokens=max_tokens, max_sequences=max_sequences)
        assert (m.ctx.room[m.buf["lists"]], m.ctx.room[m.buf["list_lens"]]) == (tokens * 12 * 4, tokens * 8)
        seqs = [m.sequence() for _ in range(max_sequences)]
        m.step(seqs, [[0] * (tokens // max_sequences)] * max_sequences, [[-1] * (tokens // max_sequences)] * max_sequences)
        m.close()


@pytest.mark.parametrize("more", [[], ["--samples", "3", "--share-prefixes"], ["--selected-pages", "66"]])
def test_the_command_takes_prompts_as_long_as_there_are_positions(monkeypatch, capsys, more):
    """... where nothing is decoded behind them; where something is, one less."""
    class Closed(HostContext):
        def close(self):
            assert not self.room

    monkeypatch.setattr(generate, "CudaContext", lambda device: Closed())
    small = ["x", "--qtype", "Q8_0", "--layers", "1", "--d-model", "64", "--heads", "2", "--kv-heads", "1", "--ffn", "64", "--vocab", "64", "--sequences", "1"]
    for prompt, tokens in ((4096, 1), (4095, 2), (7, 3)):
        monkeypatch.setattr("sys.argv", small + ["--prompt", str(prompt), "--tokens", str(tokens)] + more)
        generate.main()
        assert "tokens/s" in capsys.readouterr().out


def test_operators_refuse_gaps_ranks_and_numbers():
    """Only queries may have gaps; arrays of other ranks are refused like those of other sizes; what 32 bits do not hold is not cut down to what they do."""
    ctx = HostContext()
    gaps = lambda t: DeviceTensor(t.ptr, t.shape(), t.dtype, row_stride=int(np.prod(t.shape()[1:])) + 8)  # noqa: E731
    q, kv, table, n = dev("bf16", 3, 4, 64), dev("bf16", 9, 2, 16, 64), dev("i32", 3, 5), dev("i32", 3)
    codes, scales, lists, lens = dev("i8", 9, 2, 2, 64), dev("f32", 9, 2), dev("i32", 3, 2, 6), dev("i32", 3, 2, 2)
    gap, wrong = A.UnsupportedOperationError, ValueError

    def select(q=q, codes=codes, scales=scales, table=table, lists=lists, lens=lens, page_tokens=16, **more):
        return A.SelectPages(ctx, q, codes, scales, table, n, lists, lens, page_tokens=page_tokens, max_context=50, **more)

    assert select().args.width == 6 and select(q=gaps(q)).args.q_stride == 264
    for error, bad in ((gap, dict(codes=gaps(codes))), (gap, dict(scales=gaps(scales))), (gap, dict(table=gaps(table))), (gap, dict(lists=gaps(lists))), (gap, dict(lens=gaps(lens))),
                       (wrong, dict(lists=dev("i32", 3, 2))), (wrong, dict(lists=dev("i32", 18))), (wrong, dict(codes=dev("i8", 9))), (wrong, dict(q=dev("bf16", 3, 256))),
                       (wrong, dict(recent=2**32)), (wrong, dict(first=2**32 + 1)), (wrong, dict(max_drafts=2**32 + 1)), (wrong, dict(page_tokens=2**32 + 16))):
        with pytest.raises(error):
            select(**bad)

    def selected(q=q, lists=lists, lens=lens):
        return A.SelectedAttention(ctx, q, kv, kv, q, lists, lens)

    assert selected().args.width == 6
    for error, bad in ((gap, dict(lists=gaps(lists))), (gap, dict(lens=gaps(lens))), (wrong, dict(lists=dev("i32", 3, 2))), (wrong, dict(lists=dev("i32", 36)))):
        with pytest.raises(error):
            selected(**bad)

    def shared(table=table, **more):
        return A.SharedPrefixAttention(ctx, q, kv, kv, q, table, n, dev("i32", 2), dev("i32", 1), max_prefix=16, max_own=16, **more)

    shared()
    for error, bad in ((gap, dict(table=gaps(table))), (wrong, dict(table=dev("i32", 15))), (wrong, dict(max_drafts=2**32 + 1))):
        with pytest.raises(error):
            shared(**bad)

    cache = A.KvCache(ctx, 2, 9, 16, 2, 64)
    codes, scales = dev("i8", 2, 9, 2, 2, 64), dev("f32", 2, 9, 2)
    for bad in ((gaps(codes), scales), (codes, gaps(scales))):
        with pytest.raises(gap):
            A.PageBounds(cache, *bad)
    with pytest.raises(gap):
        A.PageBounds(cache, codes, scales).update(gaps(table), n, n, max_tokens=1)
    cache.close()


def test_bounds_that_are_closed_are_not_written():
    ctx = HostContext()
    cache = A.KvCache(ctx, 2, 9, 16, 2, 64)
    bounds = A.PageBounds(cache)
    held = len(ctx.room)
    bounds.update(dev("i32", 3, 4), dev("i32", 3), dev("i32", 3), max_tokens=1)
    for _ in range(2):
        bounds.close()
        assert len(ctx.room) == held - 2
        for call in (lambda: bounds.update(dev("i32", 3, 4), dev("i32", 3), dev("i32", 3), max_tokens=1), lambda: bounds.layer(0)):
            with pytest.raises(ValueError):
                call()
    cache.close()
