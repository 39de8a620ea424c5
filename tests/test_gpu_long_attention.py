"""Attention over lists of pages and attention of sequences that share a prefix, against the formula in 64 bits.  Tolerances as in test_gpu_attention.py: outputs are
bf16 (2^-8 of a value at most), weights are rounded to bf16 before the second product (2^-8 of sum p |v|), scores are fp32; that sums come in parts which are
joined in fp32 adds some 2^-22 of a value."""
import math

import numpy as np
import pytest

from test_gpu_attention import backend, check, formula, held, i32, normal, offsets, pages_for, tree_words  # noqa: F401

pytestmark = pytest.mark.gpu


def signed(words):
    import torch

    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device="cuda")


def same_bits(op, out, backend, times=2):
    import torch

    first = out.clone()
    for _ in range(times):
        out.fill_(7.0)
        torch.cuda.synchronize()
        op.run()
        backend.synchronize_device()
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))


# ------------------------------------------------------------------------------------------------ lists
def run_selected(backend, held_lens, news, q_heads, kv_heads, dim, page, width=None, words=None, seed=0, edit=None, pages=None, q_apart=0, heads=None):
    """held_lens[t], news[t] of every token, the same for all kv heads but one page of the context less for odd ones."""
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(seed)
    n = len(held_lens)
    lens = np.zeros((n, kv_heads, 2), np.int32)
    for t in range(n):
        for h in range(kv_heads):
            lens[t, h, 0] = max(0, held_lens[t] - (page if h & 1 else 0))
            lens[t, h, 1] = lens[t, h, 0] + news[t]
    width = width or max(1, -(-int(lens.max()) // page))
    pages = pages or 3 * width + 5
    lists = np.full((n, kv_heads, width), -1, np.int32)
    for t in range(n):
        for h in range(kv_heads):
            used = -(-int(lens[t, h, 1]) // page)
            lists[t, h, :used] = rng.permutation(pages)[:used]
    wide = normal(rng, n, (q_heads + q_apart) * dim, scale=1.5)
    q = wide[:, :q_heads * dim].unflatten(1, (q_heads, dim))
    keys, values = normal(rng, pages, kv_heads, page, dim), normal(rng, pages, kv_heads, page, dim)
    if edit:
        edit(q, keys, values, lists, lens)
    out = torch.full((n, q_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    d_lists, d_lens, scale = torch.from_numpy(lists).cuda(), torch.from_numpy(lens).cuda(), 1 / math.sqrt(dim)
    anc = signed(words) if words else None
    torch.cuda.synchronize()
    op = A.SelectedAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(d_lists), held(d_lens), ancestors=held(anc), scale=scale)
    op.run()
    backend.synchronize_device()
    same_bits(op, out, backend)
    group = q_heads // kv_heads
    for t in range(n):
        for h in heads or range(kv_heads):
            context, total = map(int, lens[t, h])
            k, v = (x[torch.from_numpy(lists[t, h, :-(-total // page)].astype(np.int64)).cuda(), h].flatten(0, 1)[:total].double().cpu() for x in (keys, values))
            seen = torch.ones(1, total, dtype=torch.bool)
            for j in range(total - context):
                seen[0, context + j] = not words or bool(words[t] >> j & 1)
            some = range(group) if group * total < 20000 else sorted({0, group - 1})
            for g in some:
                row = q[t, h * group + g][None].double().cpu()
                want, spread = formula(row, k, v, scale, seen)
                check(out[t, h * group + g][None], want, spread)
    return out


@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 1), (12, 4), (40, 2), (33, 1), (128, 1)])
def test_selected(backend, q_heads, kv_heads, dim):
    run_selected(backend, [0, 15, 16, 17, 130, 400, 33], [1, 1, 1, 1, 1, 1, 0], q_heads, kv_heads, dim, 16)


@pytest.mark.parametrize("page", [16, 64, 128, 1024])
def test_selected_pages(backend, page):
    run_selected(backend, [3 * page, page + 5, 1], [5, 1, 64], 6, 2, 96, page, width=8)


def test_selected_trees(backend):
    rng = np.random.default_rng(2)
    words = tree_words(24, rng, "tree") + tree_words(64, rng, "tree")
    run_selected(backend, [500] * 24 + [37] * 64, [24] * 24 + [64] * 64, 6, 2, 64, 16, words=words)
    run_selected(backend, [0, 16, 5], [9, 9, 9], 4, 2, 128, 16, words=[0, 0, 1 << 8])


def test_selected_rows_that_see_nothing(backend):
    import torch

    out = run_selected(backend, [0, 0, 20], [0, 4, 1], 4, 1, 64, 16, words=[5, 0, 1], width=4)
    assert torch.count_nonzero(out[:2]) == 0


def test_selected_many_lists(backend):
    """More lists than a CTA has lanes many times over, and few long ones that are cut."""
    rng = np.random.default_rng(4)
    run_selected(backend, [int(n) for n in rng.integers(0, 300, 700)], [1] * 700, 4, 2, 64, 16, pages=200)
    run_selected(backend, [9000], [3], 8, 2, 128, 64, pages=160)
    run_selected(backend, [2000] * 20, [1] * 20, 32, 8, 64, 32, pages=100, heads=[0, 7])


def test_selected_on_every_way(backend):
    """Lists by number and on a line, in clusters of large CTAs and of small ones, whole: as many lists, and of such lengths, as lead there."""
    run_selected(backend, [2100] * 76, [1] * 76, 16, 8, 64, 16, pages=140, heads=[0, 7])                    # 608 long ones: a line
    run_selected(backend, [700 + 9 * i for i in range(10)], [1] * 10, 160, 8, 128, 16, pages=140, heads=[7])   # 80 with 20 rows
    run_selected(backend, [700 + 9 * i for i in range(9)], [1] * 9, 160, 8, 128, 16, pages=140, heads=[0])
    run_selected(backend, [2100 + 9 * i for i in range(10)], [1] * 10, 160, 8, 128, 16, pages=160, heads=[7])  # longer ones, 32 rows at a time: a line
    run_selected(backend, [2100 + 9 * i for i in range(9)], [1] * 9, 160, 8, 128, 16, pages=160, heads=[0])    # clusters of 2
    run_selected(backend, [2100 + 9 * i for i in range(5)], [1] * 5, 320, 8, 64, 16, pages=160, heads=[3])     # 40 rows
    for tokens in (1, 3, 9, 12, 17, 24, 40, 60, 80):
        run_selected(backend, [1 + (37 * i) % 600 for i in range(tokens)], [1] * tokens, 16, 8, 128, 16, width=38, pages=60, heads=[0, 3])


def test_selected_one_page_many_times(backend):
    def edit(q, keys, values, lists, lens):
        lists[0, 0, :5] = [3, 3, 0, 3, 0]
        lists[1, 0, :5] = lists[0, 0, 4::-1]

    run_selected(backend, [70, 70], [3, 3], 2, 1, 64, 16, edit=edit)


def test_selected_queries_with_gaps(backend):
    run_selected(backend, [70, 200], [1, 1], 4, 2, 64, 16, q_apart=3)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_selected_unseen_keys_have_no_influence(backend, value):
    """Behind the end of a list, in pages that are not in it, and new tokens that are no ancestors; those that see it are what the formula says."""

    def edit(q, keys, values, lists, lens):
        for x in (keys, values):
            x[int(lists[0, 0, 2]), :, 8:] = value   # 37 + 3 keys: rows 8 and on of the third page
            x[int(lists[1, 0, 3]), 0, 4] = value    # place 52 of 50 + 9: new token 2
            unused = sorted(set(range(len(keys))) - set(lists[:, 0].flatten().tolist()))
            x[unused] = value

    run_selected(backend, [37, 50], [3, 9], 4, 1, 64, 16, words=[7, 0b100000011], edit=edit)
    run_selected(backend, [37, 50], [3, 9], 4, 1, 128, 16, words=[7, 0b100000111], edit=edit)


def test_selected_values_of_every_size(backend):
    def edit(q, keys, values, lists, lens):
        keys[::2] *= 1e18
        q[0] *= 1e18
        q[1] *= 1e-30

    run_selected(backend, [70, 300], [3, 9], 4, 1, 64, 16, edit=edit)


def test_selected_outside(backend):
    """Pages outside the cache are not followed, lengths that cannot be are rows of zeros; other rows keep their bits."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(3)
    q, keys, values = normal(rng, 8, 4, 64), normal(rng, 12, 2, 16, 64), normal(rng, 12, 2, 16, 64)
    lists = torch.from_numpy(rng.integers(0, 12, (8, 2, 5)).astype(np.int32)).cuda()
    lens = torch.tensor([[[60, 61], [70, 71]]] * 8, dtype=torch.int32, device="cuda")
    out, good = torch.empty_like(q), torch.empty_like(q)
    run = lambda o: A.SelectedAttention(backend.cuda_context, held(q), held(keys), held(values), held(o), held(lists), held(lens)).run()  # noqa: E731
    torch.cuda.synchronize()
    run(good)
    backend.synchronize_device()
    lists[1, 0, 2], lists[2, 1, 4], lists[3, 0, 0] = -1, 12, 2**31 - 1
    lens[4, 0], lens[5, 1], lens[6, 0], lens[7, 1] = i32([-1, 5]), i32([20, 19]), i32([3, 68]), i32([70, 81])
    torch.cuda.synchronize()
    run(out)
    with pytest.raises(N.WfError) as e:
        backend.synchronize_device()
    assert e.value.status == N.WF_ERR_INDEX
    differ = (out != good).any(-1).cpu()
    want = torch.zeros(8, 4, dtype=torch.bool)
    for t, h in ((1, 0), (2, 1), (3, 0), (4, 0), (5, 1), (6, 0), (7, 1)):
        want[t, 2 * h:2 * h + 2] = True
    assert torch.equal(differ, want)
    for t, h in ((4, 0), (5, 1), (6, 0), (7, 1)):
        assert torch.count_nonzero(out[t, 2 * h:2 * h + 2]) == 0
    # without the keys of the page that is not there
    for t, h, j in ((1, 0, 2), (2, 1, 4), (3, 0, 0)):
        total = int(lens[t, h, 1])
        kept = [i for i in range(total) if i // 16 != j]
        at = torch.tensor(kept)
        names = lists[t, h].cpu().long()[at // 16]
        k, v = (x.cpu()[names, h, at % 16].double() for x in (keys, values))
        for g in range(2):
            w, spread = formula(q[t, 2 * h + g][None].double().cpu(), k, v, 1 / 8, torch.ones(1, len(kept), dtype=torch.bool))
            check(out[t, 2 * h + g][None], w, spread)


def test_selected_refusals(backend):
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    q, keys = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(9, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    lists, lens = torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 2, dtype=torch.int32, device="cuda")

    def make(keys=keys, **more):
        return A.SelectedAttention(backend.cuda_context, held(q), held(keys), held(keys), held(torch.empty_like(q)), held(lists), held(lens), **more)

    make().run()
    backend.synchronize_device()
    for more, status in ((dict(scale=0.0), N.WF_ERR_INVALID_ARGUMENT), (dict(layer=1), N.WF_ERR_SHAPE), (dict(layer=-1), N.WF_ERR_SHAPE)):
        with pytest.raises(N.WfError) as e:
            make(**more).run()
        assert e.value.status == status
    op = make()
    op.args.width = 0
    with pytest.raises(N.WfError):
        op.run()
    with pytest.raises(ValueError):
        make(ancestors=held(lists))
    backend.synchronize_device()


# ------------------------------------------------------------------------------------------------ shared prefixes
# A bound of the prefix far above it: as much might be read again, if every sequence were to read it, that the prefixes have a kernel of their own (several = 1).  A bound of what a sequence has behind
# it as well (2): as much might lie there that its rows go 32 or 128 at a time.  Of the latter alone (3): prefixes that are known to be short.
FAR = 1 << 24


def run_shared(backend, members, prefix, own, drafts, q_heads, kv_heads, dim, page, shape="tree", seed=0, edit=None, arrays=True, only=None, most=None, garbage=False, several=False):
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(seed)
    n = sum(drafts)
    of = [g for g, m in enumerate(members) for _ in range(m)]
    q = normal(rng, n, q_heads, dim, scale=1.5)
    first = offsets(members)
    need = [-(-(a + b) // page) for a, b in zip(own, drafts)]
    order = list(rng.permutation(sum(need) + sum(p // page for p in prefix) + 2).astype(np.int32))
    pages = len(order)
    common = [[order.pop() for _ in range(p // page)] for p in prefix]
    width = max(len(common[g]) + m for g, m in zip(of, need)) or 1
    tables = np.full((len(own), width), 2**31 - 1, np.int32)
    for s, g in enumerate(of):
        row = common[g] + [order.pop() for _ in range(need[s])]
        tables[s, :len(row)] = row
        if garbage and s != first[g]:
            tables[s, :len(common[g])] = -5
    keys, values = normal(rng, pages, kv_heads, page, dim), normal(rng, pages, kv_heads, page, dim)
    words = [w for m in drafts for w in tree_words(m, rng, shape)]
    if edit:
        edit(q, keys, values, tables)
    out = torch.full((n, q_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    context = [prefix[g] + a for g, a in zip(of, own)]
    tab, ctx, off, groups, pre, scale = torch.from_numpy(tables).cuda(), i32(context), i32(offsets(drafts)), i32(first), i32(prefix), 1 / math.sqrt(dim)
    anc = signed(words) if words else torch.zeros(0, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    op = A.SharedPrefixAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(tab), held(ctx), held(groups), held(pre), max_prefix=FAR if several in (1, 2) else most or max(prefix),
                                 max_own=FAR if several >= 2 else most or max(own), q_offsets=held(off) if arrays else None, max_drafts=max(drafts), ancestors=held(anc) if arrays else None, scale=scale)
    op.run()
    backend.synchronize_device()
    same_bits(op, out, backend)
    group, starts = q_heads // kv_heads, offsets(drafts)
    for s, (g, new) in enumerate(zip(of, drafts)):
        if only and s not in only:
            continue
        total, rows = context[s] + new, slice(starts[s], starts[s + 1])
        t = np.arange(total)
        names = np.where(t < prefix[g], tables[first[g]][np.minimum(t // page, width - 1)], tables[s][t // page])
        where = torch.from_numpy(names.astype(np.int64)).cuda()
        k, v = (x[where, :, torch.from_numpy(t % page).cuda()].double().cpu() for x in (keys, values))
        seen = torch.ones(new, total, dtype=torch.bool)
        for i in range(new):
            for j in range(new):
                seen[i, context[s] + j] = bool(words[starts[s] + i] >> j & 1)
        heads = range(q_heads) if new * total * q_heads < 20000 else sorted({0, q_heads - 1})
        for h in heads:
            want, spread = formula(q[rows, h].double().cpu(), k[:, h // group], v[:, h // group], scale, seen)
            check(out[rows, h], want, spread)
    return out


several = pytest.mark.parametrize("several", [0, 1, 2, 3])


@several
@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 2), (5, 1), (40, 1), (128, 1)])
def test_shared(backend, q_heads, kv_heads, dim, several):
    run_shared(backend, [3, 1, 4], [48, 0, 160], [5, 100, 0, 33, 16, 1, 64, 7], [1] * 8, q_heads, kv_heads, dim, 16, several=several)


@several
@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("q_heads,kv_heads,dim", [(6, 2, 128), (4, 4, 64), (16, 1, 96)])
def test_shared_trees(backend, page, q_heads, kv_heads, dim, several):
    run_shared(backend, [3, 2], [page, 3 * page], [37, 200, 0, 5, 77], [9, 1, 24, 7, 3], q_heads, kv_heads, dim, page, several=several)
    run_shared(backend, [2, 1], [page, 0], [20, 3, 555], [2, 64, 5], q_heads, kv_heads, dim, page, shape="chain", garbage=True, several=several)


@several
def test_shared_few_rows(backend, several):
    """Up to 16 and 32 rows in all; prefixes in clusters and on a line; tokens of a long sequence among short ones, 32 rows at a time."""
    run_shared(backend, [2, 2], [320, 48], [5, 100, 0, 33], [1, 1, 1, 1], 8, 2, 64, 16, several=several)
    run_shared(backend, [2], [640], [5, 100], [1, 2], 20, 2, 128, 16, several=several, garbage=True)
    run_shared(backend, [2, 2, 2, 1, 1], [320, 48, 160, 0, 0], [5, 100, 0, 33, 7, 8, 9, 1], [1] * 8, 48, 16, 64, 16, several=several, only=[0, 3, 7])
    run_shared(backend, [9], [64], [5, 100, 0, 33, 7, 8, 9, 1, 60], [1, 1, 1, 12, 1, 1, 1, 1, 1], 8, 2, 64, 16, several=several)


@several
def test_shared_defaults(backend, several):
    """Without offsets and words: every sequence has max_drafts tokens, a chain; bounds far above the lengths."""
    run_shared(backend, [3, 1], [64, 16], [100, 333, 5, 0], [4, 4, 4, 4], 4, 2, 64, 16, shape="chain", arrays=False, several=several)
    run_shared(backend, [3, 1], [64, 16], [100, 333, 5, 0], [2, 4, 1, 4], 4, 2, 64, 16, most=5000)


@several
def test_shared_long_prefix(backend, several):
    """Prefixes that many CTAs take a part of, by rows that fill several tiles, one, and a few of one."""
    run_shared(backend, [40], [4096], [3 * i for i in range(40)], [1] * 40, 16, 2, 128, 64, only=[0, 17, 39], several=several)
    run_shared(backend, [2], [20000], [300, 40], [1, 1], 8, 1, 64, 32, garbage=True, several=several)
    run_shared(backend, [5, 7], [9008, 3200], [20, 700, 5, 0, 64, 3, 3, 3, 1500, 3, 3, 3], [1, 2, 1, 3, 1, 1, 1, 5, 1, 1, 1, 1], 24, 8, 64, 16, only=[0, 3, 8], several=several)


@several
def test_shared_long_own(backend, several):
    """Own contexts that are cut, behind prefixes, by few rows and by many."""
    run_shared(backend, [2, 1], [1024, 0], [9000, 10, 70], [1, 1, 1], 8, 2, 128, 64, several=several)
    run_shared(backend, [2], [512], [5000, 3000], [40, 12], 8, 2, 64, 32, garbage=True, several=several)
    run_shared(backend, [20], [64], [1500] * 10 + [30] * 10, [1] * 20, 8, 8, 64, 32, garbage=True, several=several, only=[0, 19])


@several
def test_shared_many_sequences(backend, several):
    rng = np.random.default_rng(6)
    members = [1 + int(n) for n in rng.integers(0, 7, 70)]
    count = sum(members)
    run_shared(backend, members, [16 * int(n) for n in rng.integers(0, 9, 70)], [int(n) for n in rng.integers(0, 60, count)], [1 + int(n) for n in rng.integers(0, 3, count)], 2, 1, 64, 16,
               only=list(range(0, count, 5)), several=several)


@several
def test_shared_one_long_group(backend, several):
    """More rows than two tiles: several units read the same prefix.  (On one kv head 300 sequences are few units for the SMs, on eight more than their CTAs.)"""
    run_shared(backend, [300], [256], [int(i % 40) for i in range(300)], [1] * 300, 4, 1, 64, 16, only=[0, 1, 128, 299], several=several)
    run_shared(backend, [100], [256], [int(i % 40) for i in range(100)], [1] * 100, 16, 8, 64, 16, only=[0, 1, 99], several=several)


@several
def test_shared_nothing_in_common(backend, several):
    run_shared(backend, [1, 1, 1], [0, 0, 0], [100, 333, 5], [3, 1, 2], 4, 2, 64, 16, several=several)
    run_shared(backend, [2, 1], [0, 0], [100, 333, 5], [3, 1, 2], 4, 2, 64, 16, several=several)


@several
def test_shared_rows_that_see_nothing(backend, several):
    import torch

    out = run_shared(backend, [2], [0], [0, 20], [3, 2], 4, 2, 64, 16, shape="none", several=several)
    assert torch.count_nonzero(out[:3]) == 0


@several
def test_shared_sequences_without_tokens(backend, several):
    run_shared(backend, [3, 2], [48, 32], [5, 100, 0, 33, 16], [1, 0, 2, 0, 0], 4, 2, 64, 16, several=several)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("drafts", [[2, 9, 1], [20, 9, 33]])
@several
def test_shared_unseen_keys_have_no_influence(backend, value, drafts, several):
    """Behind the ends, in drafts that are no ancestors, in another group's prefix; a row that sees it has what the formula says."""

    def edit(q, keys, values, tables):
        for x in (keys, values):
            x[int(tables[0][-(-(32 + 37 + drafts[0]) // 16) - 1]), :, (37 + drafts[0] - 1) % 16 + 1:] = value
            x[int(tables[1][(32 + 50 + 2) // 16]), 1, 4] = value  # the third draft, seen by some
            x[int(tables[2][1]), 0, 3] = value                    # the other group's prefix

    run_shared(backend, [2, 1], [32, 48], [37, 50, 9], drafts, 4, 2, 64, 16, edit=edit, garbage=True, several=several)
    run_shared(backend, [2, 1], [32, 48], [37, 50, 9], drafts, 12, 2, 128, 16, edit=edit, garbage=True, several=several)


@several
def test_shared_values_of_every_size(backend, several):
    """Scores that leave the prefix or the own keys no weight at all, near the lowest and the largest fp32."""

    def edit(q, keys, values, tables):
        keys[int(tables[0][0])] *= 1e18
        q[0] *= 1e18
        q[1] *= 1e-30
        keys[int(tables[1][3])] *= 30
        q[2:] *= 10

    run_shared(backend, [4], [48], [37, 50, 9, 16], [1, 1, 2, 1], 4, 2, 64, 16, edit=edit, several=several)
    run_shared(backend, [4], [48], [37, 50, 9, 16], [9, 11, 20, 1], 4, 2, 64, 16, edit=edit, several=several)


@several
def test_shared_outside(backend, several):
    """Groups, prefixes, contexts and pages that cannot be: reported, rows of zeros or without those keys; the others keep their bits."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(3)
    q, keys, values = normal(rng, 8, 4, 64), normal(rng, 40, 2, 16, 64), normal(rng, 40, 2, 16, 64)
    tables = torch.arange(40, dtype=torch.int32, device="cuda").repeat(8, 1)
    good_out = torch.empty_like(q)

    def run(out, tables=tables, context=(40,) * 8, groups=(0, 2, 4, 6, 8), prefix=(32,) * 4, max_prefix=FAR if several in (1, 2) else 64, max_own=40):
        tab, ctx, gr, pre = tables.contiguous(), i32(context), i32(groups), i32(prefix)
        out.fill_(7.0)
        torch.cuda.synchronize()
        A.SharedPrefixAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(tab), held(ctx), held(gr), held(pre), max_prefix=max_prefix, max_own=max_own).run()

    run(good_out)
    backend.synchronize_device()
    out = torch.empty_like(q)
    zeros = lambda: [t for t in range(8) if torch.count_nonzero(out[t]) == 0]  # noqa: E731
    same = lambda: [t for t in range(8) if torch.equal(out[t], good_out[t])]  # noqa: E731
    for bad, at in ((dict(prefix=(32, 24, 32, 32)), [2, 3]), (dict(prefix=(32, 32, -16, 32)), [4, 5]), (dict(prefix=(FAR + 16 if several in (1, 2) else 80, 32, 32, 32)), [0, 1]),
                    (dict(context=(40, 31, 40, 40, 40, 40, 73, 40)), [1, 6]), (dict(context=(40, 40, -1, 40, 40, 2**31 - 1, 40, 40)), [2, 5]),
                    (dict(groups=(1, 2, 4, 6, 8)), [0]), (dict(groups=(0, 2, 4, 6, 7)), [7]), (dict(groups=(0, 2, 4, 6, 9)), [6, 7])):
        run(out, **bad)
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX
        assert zeros() == at and same() == [t for t in range(8) if t not in at], bad
    for bad in ((0, 4, 2, 6, 8), (8, 6, 4, 2, 0), (-5, 2, 4, 6, 8)):  # which sequences are left, nothing says; no more than that
        run(out, groups=bad)
        with pytest.raises(N.WfError):
            backend.synchronize_device()
    wrong = tables.clone()
    wrong[2, 1], wrong[5, 2] = -1, 40  # of a group's prefix, of a sequence's own
    run(out, tables=wrong)
    with pytest.raises(N.WfError) as e:
        backend.synchronize_device()
    assert e.value.status == N.WF_ERR_INDEX and same() == [0, 1, 4, 6, 7]
    for t, gone in ((2, range(16, 32)), (3, range(16, 32)), (5, range(32, 48))):
        at = torch.tensor([i for i in range(41) if i not in gone])
        for h in range(4):
            k, v = (x.cpu()[at // 16, h // 2, at % 16].double() for x in (keys, values))
            w, spread = formula(q[t, h][None].double().cpu(), k, v, 1 / 8, torch.ones(1, len(at), dtype=torch.bool))
            check(out[t, h][None], w, spread)


@pytest.mark.parametrize("groups", [[0, 40] * 20, list(range(0, 41, 4)) + list(range(0, 37, 4)), list(range(0, 41, 2)) + list(range(0, 39, 2))])
def test_shared_groups_that_overlap(backend, groups):
    """More rows in groups than there are tokens: reported, and no more work than a batch that can be has (as many groups as sequences: each sequence reads for itself, and may find a group
    that it is in); the next call is as ever."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(4)
    q, keys, values = normal(rng, 40, 8, 64), normal(rng, 30, 2, 16, 64), normal(rng, 30, 2, 16, 64)
    tables, context = torch.arange(30, dtype=torch.int32, device="cuda").repeat(40, 1), i32([470] * 40)

    def run(groups):
        out, gr, pre = torch.full_like(q, 7.0), i32(groups), i32([320] * (len(groups) - 1))
        torch.cuda.synchronize()
        A.SharedPrefixAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(tables), held(context), held(gr), held(pre), max_prefix=FAR, max_own=200).run()
        return out

    good = run([0, 40])
    backend.synchronize_device()
    out = run(groups)
    with pytest.raises(N.WfError) as e:
        backend.synchronize_device()
    assert e.value.status == N.WF_ERR_INDEX and (len(groups) == 41 or torch.count_nonzero(out) == 0)
    again = run([0, 40])
    backend.synchronize_device()
    assert torch.equal(again, good)


def test_shared_is_what_trees_are(backend):
    """The same call with and without a prefix, and by TreeAttention: sums of the same products in other parts and orders.  Each is off by at most 2^-8 |out| + 2^-8 sum p |v| (check), and neither
    of these is more than the largest |v|: two results differ by at most 2 (2^-8 + 2^-8) max |v| = 2^-6 max |v|."""
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(8)
    q, keys, values = normal(rng, 6, 8, 128), normal(rng, 30, 2, 64, 128), normal(rng, 30, 2, 64, 128)
    rows = [list(range(9)) + [10 + 3 * s, 11 + 3 * s, 12 + 3 * s] for s in range(6)]
    tables, context = i32(rows), i32([9 * 64 + 20 * s for s in range(6)])
    outs = [torch.empty_like(q) for _ in range(3)]
    args = [held(x) for x in (q, keys, values)]
    torch.cuda.synchronize()
    A.TreeAttention(backend.cuda_context, *args, held(outs[0]), held(tables), held(context), max_context=700).run()
    outs.append(torch.empty_like(q))
    for out, p, most in ((outs[1], 0, 0), (outs[2], 9 * 64, 9 * 64), (outs[3], 9 * 64, FAR)):
        groups, prefix = i32([0, 6]), i32([p])
        torch.cuda.synchronize()
        A.SharedPrefixAttention(backend.cuda_context, *args, held(out), held(tables), held(context), held(groups), held(prefix), max_prefix=most, max_own=700 - p).run()
        backend.synchronize_device()
    for out in outs[1:]:
        assert (outs[0].float() - out.float()).abs().max() <= 2.0**-6 * values.float().abs().max()


def test_shared_refusals(backend):
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    q, keys = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(9, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    tables, ctx, groups, prefix = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), i32([0, 0]), i32([0, 2]), i32([0])

    def make(groups=groups, prefix=prefix, **more):
        args = dict(max_prefix=16, max_own=16) | more
        return A.SharedPrefixAttention(backend.cuda_context, held(q), held(keys), held(keys), held(torch.empty_like(q)), held(tables), held(ctx), held(groups), held(prefix), **args)

    make().run()
    backend.synchronize_device()
    for more, status in ((dict(max_prefix=-1), N.WF_ERR_SHAPE), (dict(max_own=-1), N.WF_ERR_SHAPE), (dict(max_drafts=0), N.WF_ERR_TOO_LARGE), (dict(max_drafts=65), N.WF_ERR_TOO_LARGE),
                         (dict(max_drafts=2), N.WF_ERR_SHAPE), (dict(scale=-1.0), N.WF_ERR_INVALID_ARGUMENT), (dict(groups=i32([0]), prefix=i32([])), N.WF_ERR_SHAPE),
                         (dict(groups=i32([0, 1, 2, 2]), prefix=i32([0, 0, 0])), N.WF_ERR_SHAPE)):
        with pytest.raises(N.WfError) as e:
            make(**more).run()
        assert e.value.status == status, more
    with pytest.raises(ValueError):
        make(groups=i32([0, 1, 2]))
    backend.synchronize_device()


def test_shared_and_selected_recorded(backend):
    """Recorded calls serve growing contexts, prefixes and lists; a call that would have to allocate while it is recorded is refused."""
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(11)
    ctx = backend.cuda_context
    q, keys, values = normal(rng, 3, 4, 64), normal(rng, 90, 2, 16, 64), normal(rng, 90, 2, 16, 64)
    tables = torch.arange(90, dtype=torch.int32, device="cuda").repeat(3, 1)
    context, groups, prefix = i32([0, 0, 0]), i32([0, 3]), i32([0])
    lists, lens = torch.arange(40, dtype=torch.int32, device="cuda").repeat(3, 2, 1), torch.zeros(3, 2, 2, dtype=torch.int32, device="cuda")
    outs = [torch.empty_like(q) for _ in range(4)]
    args = [held(x) for x in (q, keys, values)]
    stream = backend.create_stream()
    torch.cuda.synchronize()
    shared = A.SharedPrefixAttention(ctx, *args, held(outs[0]), held(tables), held(context), held(groups), held(prefix), max_prefix=FAR, max_own=400)
    selected = A.SelectedAttention(ctx, *args, held(outs[1]), held(lists), held(lens))
    shared.run(stream)
    ctx.synchronize(stream)
    ctx.graph_begin(stream)
    shared.run(stream)
    selected.run(stream)
    graph = ctx.graph_end(stream)
    for p, own in ((0, 3), (160, 20), (992, 400)):
        context.fill_(p + own)
        prefix.fill_(p)
        lens[..., 0], lens[..., 1] = own, own + 1
        torch.cuda.synchronize()
        ctx.graph_launch(graph, stream)
        ctx.synchronize(stream)
        A.TreeAttention(ctx, *args, held(outs[2]), held(tables), held(context), max_context=1400).run()
        short = i32([own] * 3)
        torch.cuda.synchronize()
        A.TreeAttention(ctx, *args, held(outs[3]), held(tables), held(short), max_context=640).run()
        backend.synchronize_device()
        for got, want in zip(outs, outs[2:]):
            assert (got.float() - want.float()).abs().max() <= 2.0**-6 * values.float().abs().max()  # as in test_shared_is_what_trees_are
    ctx.graph_destroy(graph)
    backend.destroy_stream(stream)


@several
def test_shared_queries_with_gaps_and_rows_behind(backend, several):
    """Tokens that lie further apart than they are long, on another stream; rows behind the last sequence stay as they were."""
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(12)
    wide = normal(rng, 5, 7 * 64)
    q, keys, values = wide[:, :4 * 64].unflatten(1, (4, 64)), normal(rng, 40, 2, 16, 64), normal(rng, 40, 2, 16, 64)
    tables, context, groups, prefix, off = torch.arange(40, dtype=torch.int32, device="cuda").repeat(3, 1), i32([70, 64, 64]), i32([0, 3]), i32([64]), i32([0, 2, 2, 3])
    out = torch.full((5, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    stream = backend.create_stream()
    torch.cuda.synchronize()
    A.SharedPrefixAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(tables), held(context), held(groups), held(prefix), max_prefix=FAR if several in (1, 2) else 64, max_own=FAR if several >= 2 else 6,
                            q_offsets=held(off), max_drafts=2).run(stream)
    backend.synchronize_stream(stream)
    assert (out[3:] == 7).all()
    for row, n in ((0, 71), (1, 72), (2, 65)):
        k, v = (x.transpose(1, 2).flatten(0, 1)[:n].double().cpu() for x in (keys, values))
        for h in range(4):
            want, spread = formula(q[row, h][None].double().cpu(), k[:, h // 2], v[:, h // 2], 1 / 8, torch.ones(1, n, dtype=torch.bool))
            check(out[row, h][None], want, spread)
    backend.destroy_stream(stream)


def test_a_step_as_it_is_used(backend):
    """Keys into the cache, bounds, selection, attention over the lists, on one stream with nothing between, three layers one after the other: every layer's attention is that of the pages that
    were selected for it."""
    import torch

    from test_gpu_select import plain_list
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(13)
    ctx, layers, pages, page, heads, dim, width = backend.cuda_context, 3, 60, 16, 2, 64, 8
    lens, drafts = [300, 100, 17], [5, 1, 3]
    n = sum(drafts)
    tables, _ = pages_for([a + b for a, b in zip(lens, drafts)], page, rng, spare=20)
    tables[tables > 1000] = 0
    cache = A.KvCache(ctx, layers, pages, page, heads, dim)
    bounds = A.PageBounds(cache)
    tab, off, context = torch.from_numpy(tables).cuda(), i32(offsets(drafts)), i32(lens)
    past = [t for m in lens for t in range(m)]
    past_slots = torch.tensor([int(tables[s][t // page]) * page + t % page for s, m in enumerate(lens) for t in range(m)], dtype=torch.int64, device="cuda")
    slots = torch.tensor([int(tables[s][(m + i) // page]) * page + (m + i) % page for s, (m, d) in enumerate(zip(lens, drafts)) for i in range(d)], dtype=torch.int64, device="cuda")
    zero, total = i32([0] * 3), i32([a + b for a, b in zip(lens, drafts)])
    outs = [torch.zeros(n, 4, dim, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]
    lists = [torch.zeros(n, heads, width, dtype=torch.int32, device="cuda") for _ in range(layers)]
    list_lens = [torch.zeros(n, heads, 2, dtype=torch.int32, device="cuda") for _ in range(layers)]
    qb = [torch.zeros(n, 4, dim, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]
    q, k, v = (torch.from_numpy(rng.standard_normal((layers, n, h, dim)).astype(np.float32)).cuda() for h in (4, heads, heads))
    pk, pv = (torch.from_numpy(rng.standard_normal((layers, len(past), heads, dim)).astype(np.float32)).cuda() for _ in range(2))
    words = signed([w for m in drafts for w in tree_words(m, rng, "tree")])
    torch.cuda.synchronize()
    for layer in range(layers):
        A.QkNormRope(ctx, None, held(pk[layer]), held(pv[layer]), None, *cache.layer(layer), None, None, slots=held(past_slots)).run()
    bounds.update(held(tab), held(zero), held(context), max_tokens=300)
    for layer in range(layers):
        keys, values = cache.layer(layer)
        A.QkNormRope(ctx, held(q[layer]), held(k[layer]), held(v[layer]), held(qb[layer]), keys, values, None, None, slots=held(slots)).run()
        A.SelectPages(ctx, held(qb[layer]), *bounds.layer(layer), held(tab), held(context), held(lists[layer]), held(list_lens[layer]), page_tokens=page, max_context=300, recent=20,
                      q_offsets=held(off), max_drafts=5, tree=True).run()
        A.SelectedAttention(ctx, held(qb[layer]), keys, values, held(outs[layer]), held(lists[layer]), held(list_lens[layer]), ancestors=held(words)).run()
    bounds.update(held(tab), held(context), held(total), max_tokens=5)
    backend.synchronize_device()

    def host(t, dtype):
        a = np.empty(t.shape(), dtype)
        ctx.copy_to_host(a, t.ptr)
        return a

    all_k, all_v = (torch.from_numpy((host(t, np.uint16).astype(np.uint32) << 16).view(np.float32)).double() for t in (cache.keys, cache.values))
    codes, scales = host(bounds.codes, np.int8).astype(np.float64), host(bounds.scales, np.float32).astype(np.float64)
    for layer in range(layers):
        for s, (m, d) in enumerate(zip(lens, drafts)):
            for i in range(d):
                row = offsets(drafts)[s] + i
                for h in range(heads):
                    got, got_lens = lists[layer][row, h].tolist(), list_lens[layer][row, h].tolist()
                    # (full pages' bounds are the same before and after the new tokens)
                    assert (got, got_lens) == plain_list(qb[layer][row, 2 * h:2 * h + 2].double().cpu().numpy(), codes[layer, :, h], scales[layer, :, h], tables[s], m, d, i, True, page, width, 1, 20)
                    t = np.arange(got_lens[1])
                    names = torch.tensor(got)[torch.from_numpy(t // page)]
                    kk, vv = all_k[layer, names, h, torch.from_numpy(t % page)], all_v[layer, names, h, torch.from_numpy(t % page)]
                    seen = torch.ones(1, len(t), dtype=torch.bool)
                    for j in range(d):
                        seen[0, got_lens[0] + j] = bool(int(words[row]) >> j & 1)
                    for g in range(2):
                        want, spread = formula(qb[layer][row, 2 * h + g][None].double().cpu(), kk, vv, 1 / 8, seen)
                        check(outs[layer][row, 2 * h + g][None], want, spread)
    bounds.close()
    cache.close()
