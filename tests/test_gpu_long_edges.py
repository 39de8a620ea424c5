"""Page bounds, selection of pages and shared prefixes where a call has just no room, numbers are at the end of their range, or offsets cannot be.  Bounds and lists are exact and
compared for equality; attention is held against 64 bits with the tolerance of test_gpu_attention.py."""
import numpy as np
import pytest

from test_gpu_attention import backend, held, i32, normal, offsets  # noqa: F401
from test_gpu_generate_long import check_bounds, closed, make
from test_gpu_long_attention import FAR, several
from test_gpu_select import bounds_of, held8, run_select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages,tokens", [(5, 24), (100, 1), (400, 24), (500, 1), (1500, 1), (1500, 8), (5000, 1), (5000, 8), (9000, 1), (9000, 8)])
def test_select_no_room_between(backend, pages, tokens):
    """Lists that have room for the pages at their ends and for none of those between: on every way that a selection goes."""
    for first, recent in ((0, 0), (1, 16)):
        width = first + (recent + tokens + 14) // 16 + 1
        rest = 16 - (recent + tokens - 2) % 16  # of a context in its last page, so that the ends are as many pages as they can be
        lens = [16 * pages + rest, 700, 0]
        run_select(backend, lens, [tokens, 1, tokens], 8, 2, 64, 16, width, first, recent, tree=True, repeat=2)
    run_select(backend, [16 * pages + 3] * (40 if pages <= 400 else 2), [1] * (40 if pages <= 400 else 2), 4, 4, 128, 16, 1, 0, 0)


@pytest.mark.parametrize("page,first,stop,most", [(1024, 1 << 30, (1 << 30) + 5, (1 << 31) - 1024), (1024, 2**31 - 2048, 2**31 - 1030, 2**31 - 2048), (1024, 5, 1030, (1 << 31) - 1024)])
def test_bounds_at_the_end_of_long_tables(backend, page, first, stop, most):
    """Tables for as many tokens as there may be, and a call with room for as many again behind the first one: its pages' numbers pass 2^31 tokens.  All but the two pages of the range
    lie outside the cache, where nothing is to be looked at."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(page)
    keys = normal(rng, 1, 3, 1, page, 8)
    codes, scales = torch.full((1, 3, 1, 2, 8), 77, dtype=torch.int8, device="cuda"), torch.full((1, 3, 1), 77.0, device="cuda")
    cache = A.KvCache(backend.cuda_context, 1, 3, page, 1, 8, keys=held(keys), values=held(keys))
    bounds = A.PageBounds(cache, held8(codes), held8(scales))
    tables = torch.full((1, 2**31 // page - 1), -7, dtype=torch.int32, device="cuda")
    tables[0, first // page], tables[0, (stop - 1) // page] = 0, 2
    at, to = i32([first]), i32([stop])
    torch.cuda.synchronize()
    bounds.update(held(tables), held(at), held(to), max_tokens=most)
    backend.synchronize_device()
    done = {2: stop - (stop - 1) // page * page}
    if first // page != (stop - 1) // page:
        done[0] = page
    for name in range(3):
        want = bounds_of(keys[0, name, 0, :done[name]]) if name in done else (np.full((2, 8), 77, np.int8), 77.0)
        assert np.array_equal(codes[0, name, 0].cpu().numpy(), want[0]) and scales[0, name, 0].item() == want[1]
    with pytest.raises(N.WfError) as e:
        bounds.update(held(tables), held(at), held(to), max_tokens=2**31)
    assert e.value.status == N.WF_ERR_SHAPE
    bounds.close()
    cache.close()


def test_bounds_of_pages_whose_drafts_are_kept_by_others():
    """Forks between step and keep: one keeps a part of a page at its place, one all of it, one moves tokens.  Bounds of full pages are those of their keys."""
    m = make(2, selected_pages=20, recent_tokens=0)
    rng = np.random.default_rng(11)
    a = m.sequence()
    m.prefill([a], [rng.integers(0, 320, 42)])
    m.step([a], [list(map(int, rng.integers(0, 320, 25)))])
    b, c = a.fork(), a.fork()
    check_bounds(m, [a, b, c])
    m.keep([a, b, c], [25] * 3, [[0, 1], list(range(25)), [0, 4, 5, 6, 7, 9]])
    assert a.pages[2] == b.pages[2] != c.pages[2] and (a.tokens, b.tokens, c.tokens) == (44, 67, 48)
    check_bounds(m, [a, b, c])
    m.step([a, b, c], [list(map(int, rng.integers(0, 320, n))) for n in (5, 1, 17)])
    m.keep([a, b, c], [5, 1, 17], [[0, 1, 2, 3], [0], [1, 2]])
    check_bounds(m, [a, b, c])
    for s in (a, b, c):
        s.free()
    closed(m)


def run_offsets(backend, offs, several, group, n, members, prefix):
    """What a call with these offsets leaves, its scratch full of another call's sums before; and what it leaves where they are one token each."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(n)
    q, keys, values = normal(rng, n, 2 * group, 64), normal(rng, 40, 2, 16, 64), normal(rng, 40, 2, 16, 64)
    groups, tables, context = i32(offsets(members)), torch.arange(40, dtype=torch.int32, device="cuda").repeat(n, 1), i32([p + 9 for p, m in zip(prefix, members) for _ in range(m)])
    pre, outs = i32(prefix), []
    for at, v in ((list(range(n + 1)), values * 1000), (list(range(n + 1)), values), (list(range(n + 1)), values * 1000), (offs, values)):
        out, off = torch.full_like(q, 7.0), i32(at)
        torch.cuda.synchronize()
        A.SharedPrefixAttention(backend.cuda_context, held(q), held(keys), held(v), held(out), held(tables), held(context), held(groups), held(pre), q_offsets=held(off), max_drafts=3,
                                max_prefix=FAR if several in (1, 2) else max(prefix), max_own=FAR if several >= 2 else 9).run()
        if at is offs:
            with pytest.raises(N.WfError) as e:
                backend.synchronize_device()
            assert e.value.status == N.WF_ERR_INDEX
        else:
            backend.synchronize_device()
        outs.append(out)
    return outs[3], outs[1]


@several
@pytest.mark.parametrize("group,members", [(2, [3, 2, 1, 2]), (4, [10, 13, 1, 16])])
def test_shared_offsets_that_cannot_be(backend, several, group, members):
    """Where a group's offsets leave the tokens, or one of its sequences has rows outside them, that group's sequences have zeros, as far as their own rows are rows; the other groups keep
    their bits, and no sum is used that this call has not made."""
    import torch

    n, first = sum(members), offsets(members)
    prefix = [160, 96, 0, 128]
    same = list(range(n + 1))
    # the last group's last offset behind the tokens; the second group's last sequence ends before it begins, and those before it lie behind the group's end
    last = same[:-1] + [n + 1]
    got, good = run_offsets(backend, last, several, group, n, members, prefix)
    assert torch.equal(got[:first[3]], good[:first[3]]) and torch.count_nonzero(got[first[3]:n - 1]) == 0 and (got[n - 1] == 7).all()
    swapped = list(same)
    swapped[first[1] + 1] = first[2] + 1  # the second group's first sequence: as many rows as reach behind its group
    if first[2] + 1 - first[1] <= 3:  # (no more than max_drafts)
        got, good = run_offsets(backend, swapped, several, group, n, members, prefix)
        others = list(range(first[1])) + list(range(first[3], n))
        assert torch.equal(got[others], good[others])
        assert torch.isfinite(got.float()).all() and got[first[1]:first[2]].float().abs().max() == 0
    before = [-1] + same[1:]
    got, good = run_offsets(backend, before, several, group, n, members, prefix)
    assert torch.equal(got[first[1]:], good[first[1]:]) and torch.count_nonzero(got[1:first[1]]) == 0 and (got[0] == 7).all()


def test_shared_prefixes_of_more_tiles_than_a_line_has(backend):
    """128 heads behind 2^28 tokens (one page, over and over) are more tiles than the CTAs' shares are counted in: reported, and no sums are used that were not made."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(21)
    q, keys, values = normal(rng, 2, 128, 8), normal(rng, 2, 128, 1024, 8), normal(rng, 2, 128, 1024, 8) * 1000
    tables = torch.zeros(2, 2**18 + 1, dtype=torch.int32, device="cuda")
    groups = i32([0, 2])

    def run(prefix):
        out, context, pre = torch.full_like(q, 7.0), i32([prefix] * 2), i32([prefix])
        torch.cuda.synchronize()
        A.SharedPrefixAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(tables), held(context), held(groups), held(pre), max_prefix=1 << 28, max_own=0).run()
        if prefix < 1 << 28:
            backend.synchronize_device()
            return out
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX
        return out

    for _ in range(2):
        assert torch.count_nonzero(run(2048)) > 0  # sums in the scratch
        assert torch.count_nonzero(run(1 << 28)) == 0


def test_selected_more_lists_than_a_line_has(backend):
    """2^27 lists, each of which is a place on the CTAs' line and 16 more for what it costs: refused before anything is read; as many as have room are done."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(22)
    tokens, few = 1 << 24, 1 << 16
    q, out, keys = (torch.empty(n, 8, 16, 8, dtype=torch.bfloat16, device="cuda") for n in (tokens // 16, tokens // 16, 1))
    q, out = q.view(tokens, 8, 8), out.view(tokens, 8, 8)
    lists, lens = torch.zeros(tokens, 8, 1, dtype=torch.int32, device="cuda"), torch.zeros(tokens, 8, 2, dtype=torch.int32, device="cuda")
    keys.copy_(normal(rng, 1, 8, 16, 8))
    lens[:few] = 1  # a key each
    out.fill_(7.0)
    torch.cuda.synchronize()
    with pytest.raises(N.WfError) as e:
        A.SelectedAttention(backend.cuda_context, held(q), held(keys), held(keys), held(out), held(lists), held(lens)).run()
    assert e.value.status == N.WF_ERR_TOO_LARGE
    backend.synchronize_device()
    assert (out == 7).all()
    q[:few] = normal(rng, few, 8, 8)
    torch.cuda.synchronize()
    A.SelectedAttention(backend.cuda_context, held(q[:few]), held(keys), held(keys), held(out[:few]), held(lists[:few]), held(lens[:few])).run()
    backend.synchronize_device()
    assert torch.equal(out[:few], keys[0, :, 0].expand(few, 8, 8)) and (out[few:] == 7).all()


def test_shared_sums_of_no_more_than_a_call_may_have(backend):
    """Rows whose sums over a prefix would take more than 1 GiB: the call does without, in far less memory.  Both it and the one beside it, with fewer rows, are what TreeAttention
    gives, to 2^-6 of the largest value (as in test_shared_is_what_trees_are)."""
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(23)
    heads, dim, drafts = 128, 72, 64
    keys, values = normal(rng, 600, 1, 32, dim), normal(rng, 600, 1, 32, dim)
    groups, prefix = None, i32([64])
    for seqs in (254, 200):
        n = seqs * drafts
        assert (n * heads * 130 * 4 > 1 << 30) == (seqs == 254)
        q = torch.randn(n, heads, dim, device="cuda", dtype=torch.bfloat16, generator=torch.Generator(device="cuda").manual_seed(seqs))
        tables, context, groups = i32([[0, 1, 2 + 2 * s, 3 + 2 * s] for s in range(seqs)]), i32([64] * seqs), i32([0, seqs])
        want, out = torch.empty_like(q), torch.full_like(q, 7.0)
        args = [held(x) for x in (q, keys, values)]
        torch.cuda.synchronize()
        A.TreeAttention(backend.cuda_context, *args, held(want), held(tables), held(context), max_context=64, max_drafts=drafts).run()
        backend.synchronize_device()
        free = torch.cuda.mem_get_info()[0]
        A.SharedPrefixAttention(backend.cuda_context, *args, held(out), held(tables), held(context), held(groups), held(prefix), max_prefix=64, max_own=0, max_drafts=drafts).run()
        backend.synchronize_device()
        if seqs == 254:
            assert free - torch.cuda.mem_get_info()[0] < 256 << 20
        assert (out.float() - want.float()).abs().max() <= 2.0**-6 * values.float().abs().max()
