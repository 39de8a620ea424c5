"""Bounds of the keys of pages and the selection of pages by them, against plain forms in 64 bits.  Both are exact: codes are whole numbers that the definition fixes, scores whole
numbers times powers of two, so everything is compared for equality."""
import math

import numpy as np
import pytest

from test_gpu_attention import backend, held, i32, normal, offsets, pages_for  # noqa: F401

pytestmark = pytest.mark.gpu


def held8(t):
    import torch

    from warpforge_b200.backend import DeviceTensor

    return DeviceTensor(t.data_ptr(), tuple(t.shape), "i8", owner=t) if t.dtype == torch.int8 else held(t)


def least_exponent(size):
    e = -60
    while size > 127 * 2.0**e:
        e += 1
    return e


def bounds_of(keys):
    """codes [2, dim] and scale of keys [tokens, dim] in 64 bits."""
    k = keys.double().cpu().numpy()
    if not np.isfinite(k).all():
        return np.zeros((2, k.shape[1]), np.int8), math.inf
    step = 2.0 ** least_exponent(np.abs(k).max())
    return np.stack((np.ceil(k.max(0) / step), np.floor(k.min(0) / step))).astype(np.int8), step


def run_bounds(backend, lens, new, layers, heads, dim, page, seed=0, edit=None, most=None, stream=0):
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(seed)
    tables, pages = pages_for(lens, page, rng)
    keys, values = normal(rng, layers, pages, heads, page, dim), normal(rng, layers, pages, heads, page, dim)
    if edit:
        edit(keys, tables)
    codes = torch.full((layers, pages, heads, 2, dim), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((layers, pages, heads), 77.0, device="cuda")
    want_codes, want_scales = codes.cpu().numpy().copy(), scales.cpu().numpy().copy()
    for s, (n, m) in enumerate(zip(lens, new)):
        for j in range((n - m) // page, -(-n // page)) if m else ():
            name = int(tables[s][j])
            for layer in range(layers):
                for h in range(heads):
                    want_codes[layer, name, h], want_scales[layer, name, h] = bounds_of(keys[layer, name, h, :min(page, n - j * page)])
    cache = A.KvCache(backend.cuda_context, layers, pages, page, heads, dim, keys=held(keys), values=held(values))
    bounds = A.PageBounds(cache, held8(codes), held8(scales))
    tab, first, stop = torch.from_numpy(tables).cuda(), i32([n - m for n, m in zip(lens, new)]), i32(lens)
    torch.cuda.synchronize()
    bounds.update(held(tab), held(first), held(stop), max_tokens=max(new) if most is None else most, stream=stream)
    backend.synchronize_stream(stream)
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    got_codes, got_scales = bounds.layer(layers - 1)
    assert got_codes.ptr == codes[layers - 1].data_ptr() and got_scales.ptr == scales[layers - 1].data_ptr() and got_codes.shape() == (pages, heads, 2, dim)
    bounds.close()
    cache.close()


@pytest.mark.parametrize("dim", [8, 16, 24, 64, 72, 80, 96, 112, 120, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_bounds(backend, dim, page):
    run_bounds(backend, [1, page, page + 1, 0, 3 * page - 1, 700], [1, page, 1, 0, 2 * page, 700], 2, 3, dim, page)


def test_bounds_of_a_step(backend):
    run_bounds(backend, [1 + 17 * i for i in range(40)], [1] * 40, 5, 2, 128, 64)


def test_bounds_with_room_for_more(backend):
    run_bounds(backend, [100, 40], [3, 40], 1, 2, 64, 16, most=200)


def test_bounds_on_another_stream(backend):
    s = backend.create_stream()
    run_bounds(backend, [100, 40], [3, 40], 2, 2, 64, 16, stream=s)
    backend.destroy_stream(s)


def test_bounds_of_odd_values(backend):
    """Every size of a power of two and those next to it, zeros, the smallest and the largest numbers, Inf and NaN; what lies behind the last token does not count."""
    import torch

    tiny = torch.finfo(torch.bfloat16).smallest_normal

    def edit(keys, tables):
        name = lambda j: int(tables[0][j])  # noqa: E731
        keys[:, name(0)] = 0
        keys[0, name(1)] *= 2.0**-130
        keys[0, name(2)] = torch.finfo(torch.bfloat16).max
        keys[0, name(3), 0, 5, 7] = float("nan")
        keys[0, name(3), 1, 5, 7] = float("inf")
        keys[1, name(3), 0, 15, 63] = -float("inf")
        for i in range(16):
            keys[0, name(4), 0, i] = keys[0, name(4), 0, i].clamp(-1, 1)
        keys[0, name(4), 0, 3, 9] = 127 / 64  # 127 x 2^-6: the largest of a scale
        keys[1, name(4), 0, 3, 9] = 255 / 32  # the next one needs the next scale
        keys[1, name(5), 0] = -tiny
        keys[:, name(6), :, 4:] = float("nan")  # 100 = 6 x 16 + 4 tokens

    run_bounds(backend, [100], [100], 2, 2, 64, 16, edit=edit)


def test_bounds_outside(backend):
    """A page outside the cache, a range that cannot be or is longer than was said: reported and left out; the others are done."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(1)
    keys = normal(rng, 1, 6, 2, 16, 64)
    codes, scales = torch.full((1, 6, 2, 2, 64), 77, dtype=torch.int8, device="cuda"), torch.full((1, 6, 2), 77.0, device="cuda")
    cache = A.KvCache(backend.cuda_context, 1, 6, 16, 2, 64, keys=held(keys), values=held(keys))
    bounds = A.PageBounds(cache, held8(codes), held8(scales))
    tables = i32([[0, 6], [1, -1], [2, 3], [4, 5], [5, 5]])
    first, stop = i32([0, 0, 17, -1, 0]), i32([32, 32, 32, 10, 33])
    torch.cuda.synchronize()
    bounds.update(held(tables), held(first), held(stop), max_tokens=32)
    with pytest.raises(N.WfError) as e:
        backend.synchronize_device()
    assert e.value.status == N.WF_ERR_INDEX
    done = (scales != 77).cpu()[0, :, 0].tolist()
    assert done == [True, True, False, True, False, False]
    assert ((codes != 77).cpu().any(-1).any(-1).any(-1)[0].tolist()) == done
    first, stop = i32([0] * 5), i32([32, 0, 0, 0, 0])
    torch.cuda.synchronize()
    bounds.update(held(tables), held(first), held(stop), max_tokens=16)  # up to two pages: as long as the pages are not more, it is done
    with pytest.raises(N.WfError):
        backend.synchronize_device()
    cache.close()


def test_bounds_refusals(backend):
    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    import torch

    ctx, keys = backend.cuda_context, torch.zeros(2, 4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    codes, scales = torch.zeros(2, 4, 2, 2, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 4, 2, device="cuda")
    cache = A.KvCache(ctx, 2, 4, 16, 2, 64, keys=held(keys), values=held(keys))
    bounds = A.PageBounds(cache, held8(codes), held8(scales))
    tab, n = i32([[0, 1]]), i32([3])
    for more in (dict(max_tokens=-1), dict(max_tokens=1 << 31)):
        with pytest.raises(N.WfError) as e:
            bounds.update(held(tab), held(n), held(n), **more)
        assert e.value.status == N.WF_ERR_SHAPE
    bounds.update(held(tab), held(n), held(n), max_tokens=0)
    own = A.PageBounds(cache)
    own.update(held(tab), held(i32([0])), held(n), max_tokens=3)
    backend.synchronize_device()
    own.close()
    own.close()
    cache.close()


# ------------------------------------------------------------------------------------------------ selection
def plain_list(q, codes, scales, table, context, rows, place, tree, page, width, first, recent):
    """One token and kv head: q [group, dim], codes [pages, 2, dim], scales [pages] in 64 bits."""
    last, tail = -(-(context + rows) // page), max(0, context - recent) // page
    first = min(first, tail)
    between = tail - first
    k = min(between, width - first - (last - tail))
    q8 = np.zeros_like(q)
    for h in range(len(q)):
        if np.isfinite(q[h]).all():
            step = 2.0 ** least_exponent(np.abs(q[h]).max())
            q8[h] = np.rint(q[h] / step) * step
    score = []
    for p in range(first, tail):
        name = table[p]
        if not 0 <= name < len(scales):
            score.append(-math.inf)
        elif math.isinf(scales[name]):
            score.append(math.inf)
        else:
            score.append((q8 * np.where(q8 > 0, codes[name, 0], codes[name, 1]) * scales[name]).sum(-1).max())
    best = sorted(sorted(range(between), key=lambda p: (-score[p], p))[:k])
    which = list(range(first)) + [first + p for p in best] + list(range(tail, last))
    held_ = context - page * (between - k)
    return [int(table[p]) for p in which] + [-1] * (width - len(which)), [held_, held_ + (rows if tree else place + 1)]


def run_select(backend, lens, drafts, q_heads, kv_heads, dim, page, width, first=1, recent=0, tree=False, seed=0, edit=None, arrays=True, most=None, spread=30, repeat=1, q_apart=0):
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(seed)
    n = sum(drafts)
    q = normal(rng, n, (q_heads + q_apart) * dim, scale=1.5)[:, :q_heads * dim].unflatten(1, (q_heads, dim))
    tables, pages = pages_for([a + b for a, b in zip(lens, drafts)], page, rng)
    middle, half = rng.integers(-spread, spread + 1, (pages, kv_heads, 1, dim)), rng.integers(0, 128 - spread, (pages, kv_heads, 1, dim))
    codes = torch.from_numpy(np.concatenate((middle + half, middle - half), 2).clip(-127, 127).astype(np.int8)).cuda()
    scales = torch.from_numpy((2.0 ** rng.integers(-7, -4, (pages, kv_heads))).astype(np.float32)).cuda()
    if edit:
        edit(q, codes, scales, tables)
    out, out_lens = torch.full((n, kv_heads, width), 99, dtype=torch.int32, device="cuda"), torch.full((n, kv_heads, 2), 99, dtype=torch.int32, device="cuda")
    tab, ctx, off = torch.from_numpy(tables).cuda(), i32(lens), i32(offsets(drafts))
    torch.cuda.synchronize()
    op = A.SelectPages(backend.cuda_context, held(q), held8(codes), held8(scales), held(tab), held(ctx), held(out), held(out_lens), page_tokens=page, max_context=most or max(lens),
                       first=first, recent=recent, q_offsets=held(off) if arrays else None, max_drafts=max(drafts), tree=tree)
    for _ in range(repeat):
        op.run()
    backend.synchronize_device()
    group, starts = q_heads // kv_heads, offsets(drafts)
    want, want_lens = np.full(out.shape, 99, np.int32), np.full(out_lens.shape, 99, np.int32)
    q64, c64, s64 = q.double().cpu().numpy(), codes.double().cpu().numpy(), scales.double().cpu().numpy()
    for s, (context, rows) in enumerate(zip(lens, drafts)):
        for i in range(rows):
            for h in range(kv_heads):
                want[starts[s] + i, h], want_lens[starts[s] + i, h] = plain_list(q64[starts[s] + i, h * group:(h + 1) * group], c64[:, h], s64[:, h], tables[s], context, rows, i, tree,
                                                                                 page, width, first, recent)
    assert np.array_equal(out_lens.cpu().numpy(), want_lens)
    got = out.cpu().numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    return got


@pytest.mark.parametrize("dim", [8, 64, 72, 80, 96, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 2), (9, 1), (20, 4), (128, 1)])
def test_select(backend, q_heads, kv_heads, dim):
    run_select(backend, [0, 1, 16, 17, 500, 999, 333], [1] * 7, q_heads, kv_heads, dim, 16, 12)


@pytest.mark.parametrize("page", [16, 128, 1024])
@pytest.mark.parametrize("first,recent,width", [(0, 0, 3), (1, 1, 7), (4, 130, 24), (7, 16, 300)])
def test_select_ends(backend, page, first, recent, width):
    if width < first + (recent + 9 + page - 2) // page + 1:
        width += 20
    run_select(backend, [40 * page, 3 * page, 5, 0, 17 * page - 1, 9 * page + 1], [9, 1, 4, 9, 0, 3], 4, 2, 64, page, width, first, recent, tree=True)
    run_select(backend, [40 * page, 3 * page, 5, 0, 17 * page - 1, 9 * page + 1], [9, 1, 4, 9, 0, 3], 4, 2, 64, page, width, first, recent)


@pytest.mark.parametrize("pages", [255, 256, 257, 511, 512, 513, 1024, 2047, 5000])
def test_select_long(backend, pages):
    """Both sides of where a token's pages are scored by several CTAs, and the threads' runs of pages."""
    run_select(backend, [16 * pages + 3], [1], 8, 2, 64, 16, 40, repeat=3)
    run_select(backend, [16 * pages], [2], 4, 1, 128, 16, pages // 2, repeat=2)


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(4, 4, 64), (8, 4, 128), (12, 4, 96), (28, 4, 8), (48, 4, 72)])
def test_select_many_tokens(backend, q_heads, kv_heads, dim):
    """As many scores as have a kernel of their own, with groups of 1, 2, 3, 7 and 12 heads; a sequence with few pages and one without a context among them."""
    run_select(backend, [16 * 600 + 5, 700, 0, 300], [20, 3, 9, 0], q_heads, kv_heads, dim, 16, 30, tree=True, repeat=2)


@pytest.mark.parametrize("pages,tokens", [(1500, 12), (8150, 8), (8200, 8), (9000, 1)])
def test_select_many_pages(backend, pages, tokens):
    """Runs of pages in registers and, where there are more, in shared memory."""
    run_select(backend, [16 * pages + 3], [tokens], 8, 4 if pages == 1500 else 1, 64, 16, 100)


def test_select_most_pages(backend):
    """As many pages as a call may have, by as many heads as a group may have; one more is refused."""
    from warpforge_b200 import _native as N

    run_select(backend, [16 * N.WF_SELECT_MAX_PAGES], [1], 128, 1, 8, 16, 60)
    run_select(backend, [16 * N.WF_SELECT_MAX_PAGES], [2], 2, 1, 128, 16, 60)
    with pytest.raises(N.WfError) as e:
        run_select(backend, [16 * N.WF_SELECT_MAX_PAGES + 1], [1], 2, 1, 8, 16, 60)
    assert e.value.status == N.WF_ERR_TOO_LARGE


@pytest.mark.parametrize("group,dim", [(1, 8), (2, 128), (3, 96), (4, 64), (7, 72), (12, 80)])
def test_select_many_tokens_of_many_sequences(backend, group, dim):
    """Trees of so many sequences that their scores have a kernel of their own, in groups of all widths, with tokens in several parts."""
    rng = np.random.default_rng(group)
    drafts = [24] * 9 + [1, 0, 7, 24]
    run_select(backend, [int(n) for n in rng.integers(300, 16 * 60, 13)], drafts, 8 * group, 8, dim, 16, 12, tree=True)


@pytest.mark.parametrize("pages", [520, 2040, 2060, 8150, 8200])
def test_select_long_runs_of_several_tokens(backend, pages):
    run_select(backend, [16 * pages + 3, 700], [8, 7], 2, 2, 64, 16, 60, repeat=2)
    if pages < 2100:
        run_select(backend, [16 * pages, 16 * pages - 100], [13, 12], 10, 2, 128, 16, 30)


@pytest.mark.parametrize("pages", [3, 100, 128, 129, 400, 512])
@pytest.mark.parametrize("what", ["scores", "ties", "one", "odd"])
def test_select_many_lists_of_few_pages(backend, pages, what):
    """Lists that a warp has, with contexts from none to `pages` pages: scores of all sizes, of two sizes, all alike, and pages that come before all others or are nowhere."""
    rng = np.random.default_rng(pages)

    def edit(q, codes, scales, tables):
        if what in ("ties", "one"):
            codes[:] = codes[0, 0, 0, 0]
            scales[:] = 0.25
        if what == "ties":
            scales[::3] = 0.5
        if what == "odd":
            scales[::5] = float("inf")
            q[::7, 1] = float("nan")
            q[::11] = 0.0

    lens = [16 * pages] + [int(n) for n in rng.integers(0, 16 * pages + 1, 10)]
    drafts = [24] + [int(n) for n in rng.integers(0, 25, 10)]
    run_select(backend, lens, drafts, 16, 8, 64, 16, 11 + pages // 9, first=2, recent=20, tree=True, edit=edit, most=16 * max(pages, 500 if pages > 128 else 120), repeat=2)
    run_select(backend, [16 * pages] * 40, [24] * 40, 2, 1, 8, 16, 9, edit=edit, arrays=False, most=16 * max(pages, 500 if pages > 128 else 120))


def test_select_ties_of_many_tokens(backend):
    def two(q, codes, scales, tables):
        codes[:] = codes[0, 0, 0, 0]
        scales[:] = 0.25
        scales[::3] = 0.5

    run_select(backend, [16 * 1100], [16], 8, 4, 64, 16, 50, edit=two)
    run_select(backend, [16 * 1100], [16], 8, 4, 64, 16, 700, edit=two)


def test_select_batch(backend):
    rng = np.random.default_rng(7)
    run_select(backend, [int(n) for n in rng.integers(0, 9000, 60)], [1] * 60, 16, 4, 128, 64, 20, 1, 128)


def test_select_defaults_and_gaps(backend):
    """Every sequence has max_drafts tokens; queries lie further apart than they are long; the bound of the context is far above it."""
    run_select(backend, [900, 300], [3, 3], 8, 2, 64, 16, 9, arrays=False, q_apart=2, most=4000)


def test_select_ties(backend):
    """Pages of one score: the earliest are taken, however many there are of it."""

    def same(q, codes, scales, tables):
        codes[:] = codes[0, 0, 0, 0]
        scales[:] = 0.25

    run_select(backend, [3000], [1], 4, 2, 64, 16, 50, edit=same)

    def two(q, codes, scales, tables):
        same(q, codes, scales, tables)
        scales[::3] = 0.5

    run_select(backend, [3000], [1], 4, 2, 64, 16, 50, edit=two)
    run_select(backend, [3000], [1], 4, 2, 64, 16, 100, edit=two)

    def zeros(q, codes, scales, tables):
        q[:] = 0
        q[:, 1] = -q[:, 1]

    run_select(backend, [3000], [1], 4, 2, 64, 16, 50, edit=zeros)


def test_select_odd_values(backend):
    """Pages of the scale Inf come first; heads that are not finite score 0; queries of every size; pages outside the cache come last and are reported."""
    import torch

    from warpforge_b200 import _native as N

    def odd(q, codes, scales, tables):
        scales[int(tables[0][7])] = float("inf")
        scales[int(tables[0][90])] = float("inf")
        q[0, 0, 3] = float("nan")
        q[0, 1] = float("inf")
        q[1, 2:] *= 1e-30
        q[2] *= 1e20
        q[2, 5] = -torch.finfo(torch.bfloat16).max

    run_select(backend, [2000], [3], 8, 2, 64, 16, 20, edit=odd)

    def outside(q, codes, scales, tables):
        tables[0][5], tables[0][60], tables[0][61] = -1, 2**31 - 1, len(scales)

    with pytest.raises(N.WfError) as e:
        run_select(backend, [2000], [3], 8, 2, 64, 16, 20, edit=outside)
    assert e.value.status == N.WF_ERR_INDEX


def test_select_sequences_that_cannot_be(backend):
    """A context that is negative or longer than was said: empty lists; offsets that cannot be: nothing; rows behind the last sequence stay as they were."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(3)
    q, codes, scales = normal(rng, 5, 2, 64), torch.zeros(40, 1, 2, 64, dtype=torch.int8, device="cuda"), torch.ones(40, 1, device="cuda")
    tables = torch.arange(40, dtype=torch.int32, device="cuda").repeat(4, 1)
    out, lens = torch.full((5, 1, 6), 99, dtype=torch.int32, device="cuda"), torch.full((5, 1, 2), 99, dtype=torch.int32, device="cuda")
    ctx, off = i32([-1, 600, 321, 20]), i32([0, 1, 2, 3, 2])
    torch.cuda.synchronize()
    A.SelectPages(backend.cuda_context, held(q), held8(codes), held8(scales), held(tables), held(ctx), held(out), held(lens), page_tokens=16, max_context=599, recent=0, q_offsets=held(off)).run()
    with pytest.raises(N.WfError) as e:
        backend.synchronize_device()
    assert e.value.status == N.WF_ERR_INDEX
    assert out[:2].eq(-1).all() and lens[:2].eq(0).all() and out[2, 0].tolist() == [0, 1, 2, 3, 4, 20] and lens[2, 0].tolist() == [81, 82] and out[3:].eq(99).all() and lens[3:].eq(99).all()


def test_select_refusals(backend):
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    q, codes, scales = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(9, 2, 2, 64, dtype=torch.int8, device="cuda"), torch.zeros(9, 2, device="cuda")
    tables, ctx = torch.zeros(2, 9, dtype=torch.int32, device="cuda"), i32([0, 0])

    def make(width=8, **more):
        args = dict(page_tokens=16, max_context=100, recent=16) | more
        out, lens = torch.zeros(2, 2, width, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 2, dtype=torch.int32, device="cuda")
        return A.SelectPages(backend.cuda_context, held(q), held8(codes), held8(scales), held(tables), held(ctx), held(out), held(lens), **args)

    make().run()
    backend.synchronize_device()
    make(width=4).run()  # 1 + (16 + 1 + 14) / 16 + 1 = 3
    for more, status in ((dict(width=2), N.WF_ERR_SHAPE), (dict(page_tokens=24), N.WF_ERR_SHAPE), (dict(page_tokens=8), N.WF_ERR_SHAPE), (dict(first=-1), N.WF_ERR_SHAPE),
                         (dict(recent=-1), N.WF_ERR_SHAPE), (dict(first=7), N.WF_ERR_SHAPE), (dict(max_drafts=0), N.WF_ERR_TOO_LARGE), (dict(max_drafts=65), N.WF_ERR_TOO_LARGE),
                         (dict(max_drafts=2), N.WF_ERR_SHAPE), (dict(max_context=-1), N.WF_ERR_SHAPE)):
        with pytest.raises(N.WfError) as e:
            make(**more).run()
        assert e.value.status == status, more
    backend.synchronize_device()


def test_select_replayed(backend):
    """A recorded selection serves a growing context."""
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(9)
    ctx = backend.cuda_context
    q = normal(rng, 1, 8, 64)
    codes = torch.from_numpy(rng.integers(-60, 60, (64, 2, 2, 64)).astype(np.int8)).cuda()
    scales = torch.ones(64, 2, device="cuda")
    tables, lens_in = torch.arange(64, dtype=torch.int32, device="cuda")[None], i32([0])
    out, lens = torch.zeros(1, 2, 9, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, 2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    op = A.SelectPages(ctx, held(q), held8(codes), held8(scales), held(tables), held(lens_in), held(out), held(lens), page_tokens=16, max_context=1000, recent=16)
    stream = backend.create_stream()
    ctx.graph_begin(stream)
    op.run(stream)
    graph = ctx.graph_end(stream)
    for n in (5, 100, 160, 1000):
        lens_in.fill_(n)
        torch.cuda.synchronize()
        ctx.graph_launch(graph, stream)
        ctx.synchronize(stream)
        for h in range(2):
            want = plain_list(q[0, 4 * h:4 * h + 4].double().cpu().numpy(), codes[:, h].double().cpu().numpy(), scales[:, h].double().cpu().numpy(), list(range(64)), n, 1, 0, False, 16, 9, 1, 16)
            assert (out[0, h].tolist(), lens[0, h].tolist()) == want
    ctx.graph_destroy(graph)
    backend.destroy_stream(stream)


def test_select_of_several_tokens_recorded(backend):
    """Scores of several tokens lie in the scratch of the stream: it has to be there before the call is recorded; replayed beside a larger call on the same stream the graph keeps its own."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(13)
    ctx = backend.cuda_context

    def make(tokens, pages, most):
        q = normal(rng, tokens, 4, 64)
        codes, scales = torch.from_numpy(rng.integers(-60, 60, (pages, 2, 2, 64)).astype(np.int8)).cuda(), torch.ones(pages, 2, device="cuda")
        tables, context = torch.arange(pages, dtype=torch.int32, device="cuda")[None], i32([0])
        out, lens = torch.zeros(tokens, 2, 20, dtype=torch.int32, device="cuda"), torch.zeros(tokens, 2, 2, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        op = A.SelectPages(ctx, held(q), held8(codes), held8(scales), held(tables), held(context), held(out), held(lens), page_tokens=16, max_context=most, recent=16, max_drafts=tokens, tree=True)
        return op, q, codes, scales, context, out, lens

    op, q, codes, scales, context, out, lens = make(24, 2000, 16 * 1990)
    larger = make(24, 4000, 16 * 3990)
    stream = backend.create_stream()
    ctx.graph_begin(stream)
    with pytest.raises(N.WfError) as e:
        op.run(stream)
    assert e.value.status == N.WF_ERR_RECORDING
    ctx.graph_destroy(ctx.graph_end(stream))
    op.run(stream)
    ctx.graph_begin(stream)
    op.run(stream)
    graph = ctx.graph_end(stream)
    larger[0].run(stream)
    for n in (5, 600, 16 * 1990):
        context.fill_(n)
        torch.cuda.synchronize()
        ctx.graph_launch(graph, stream)
        larger[0].run(stream)
        ctx.synchronize(stream)
        for t in (0, 23):
            for h in range(2):
                want = plain_list(q[t, 2 * h:2 * h + 2].double().cpu().numpy(), codes[:, h].double().cpu().numpy(), scales[:, h].double().cpu().numpy(), list(range(2000)), n, 24, t, True, 16, 20, 1, 16)
                assert (out[t, h].tolist(), lens[t, h].tolist()) == want
    ctx.graph_destroy(graph)
    backend.destroy_stream(stream)
