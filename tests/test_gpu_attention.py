"""Attention over packed prompts and over a paged cache against the formulas in 64 bits, at the sizes and masks where kernels go wrong.

Tolerances.  Outputs are bf16, eight bits of significand: a rounded result is off by at most 2^-8 of itself.  The kernels round the weights to
bf16 before the second product: each is off by at most 2^-8 of itself, so the sum by at most 2^-8 sum_t p_t |v_t|, which `spread` below is.  Scores come from exact products summed in fp32 (dim <= 128 terms: 128 * 2^-24 of the sum of their magnitudes,
which stays below 2^-11 of a weight for the inputs here, |scale q k| summed <= 64).  Together |error| <= 2^-8 |out| + 2^-8 spread + 1e-6, spread = sum p |v|."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    from warpforge_b200.backend import NvidiaBackend

    b = NvidiaBackend(0)
    yield b
    b.close()


def held(t):
    import torch

    from warpforge_b200.backend import DeviceTensor

    if t is None:
        return None
    names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.int32: "i32", torch.int64: "i64"}
    return DeviceTensor(t.data_ptr(), tuple(t.shape), names[t.dtype], owner=t, row_stride=t.stride(0) if t.dim() == 3 else 0)


def i32(values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets(lens):
    return [0] + list(np.cumsum(lens))


def pages_for(totals, page, rng, spare=2):
    need = [-(-n // page) for n in totals]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    tables = np.full((len(totals), max(1, max(need))), 2**31 - 1, np.int32)  # what lies behind a sequence's pages is not looked at
    at = 0
    for row, n in zip(tables, need):
        row[:n] = order[at:at + n]
        at += n
    return tables, sum(need) + spare


def formula(q, k, v, scale, seen):
    """out and spread [rows, dim] in 64 bits; keys that a row does not see count for nothing whatever they hold."""
    import torch

    out, spread = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64), torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    for i in range(q.shape[0]):
        idx = torch.nonzero(seen[i]).flatten()
        if len(idx) == 0:
            continue
        s = (k[idx] @ q[i]) * scale
        p = torch.softmax(s, 0)
        out[i], spread[i] = p @ v[idx], p @ v[idx].abs()
    return out, spread


def check(got, want, spread):
    import torch

    got = got.double().cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = ~nan & ~inf
    assert torch.isfinite(got[fine]).all()
    bound = 2.0**-8 * want.abs() + 2.0**-8 * spread + 1e-6
    off = (got - want).abs()[fine]
    assert (off <= bound[fine]).all(), f"worst {float((off / bound[fine]).max()):.3g} of the bound"


def normal(rng, *shape, scale=1.0):
    import torch

    return torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).bfloat16().cuda()


def run_prompt(backend, lens, q_heads, kv_heads, dim, page=0, past=None, seed=0, q_apart=0, edit=None):
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(seed)
    n = sum(lens)
    wide = normal(rng, n, (q_heads + q_apart) * dim, scale=1.5)
    q = wide[:, :q_heads * dim].unflatten(1, (q_heads, dim))
    totals = [a + b for a, b in zip(lens, past)] if past else list(lens)
    tables = None
    if page:
        tables, pages = pages_for(totals, page, rng)
        keys, values = normal(rng, pages, kv_heads, page, dim), normal(rng, pages, kv_heads, page, dim)
    else:
        keys, values = normal(rng, n, kv_heads, dim), normal(rng, n, kv_heads, dim)
    if edit:
        edit(q, keys, values, tables)
    out = torch.full((n, q_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    tab = torch.from_numpy(tables).cuda() if page else None
    off, k_lens, scale = i32(offsets(lens)), i32(totals) if page else None, 1 / math.sqrt(dim)
    torch.cuda.synchronize()
    op = A.PromptAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(off), tables=held(tab), k_lens=held(k_lens), scale=scale)
    op.run()
    backend.synchronize_device()
    group = q_heads // kv_heads
    starts = offsets(lens)
    for s, (new, total) in enumerate(zip(lens, totals)):
        rows = slice(starts[s], starts[s + 1])
        if page:
            t = np.arange(total)
            where = torch.from_numpy(tables[s][t // page].astype(np.int64)).cuda() if total else torch.zeros(0, dtype=torch.int64, device="cuda")
            at = torch.from_numpy(t % page).cuda()
            k, v = keys[where, :, at].double().cpu(), values[where, :, at].double().cpu()
        else:
            k, v = keys[rows].double().cpu(), values[rows].double().cpu()
        seen = torch.arange(total)[None, :] <= torch.arange(new)[:, None] + (total - new)
        heads = range(q_heads) if new * total < 40000 else sorted({0, q_heads - 1, q_heads // 2})
        for h in heads:
            want, spread = formula(q[rows, h].double().cpu(), k[:, h // group], v[:, h // group], scale, seen)
            check(out[rows, h], want, spread)
    return out


@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (4, 2), (6, 2), (5, 1), (16, 1)])
def test_prompt_packed(backend, q_heads, kv_heads, dim):
    run_prompt(backend, [1, 129, 0, 40, 256], q_heads, kv_heads, dim)


@pytest.mark.parametrize("lens", [[1], [127], [128], [129], [255], [257], [383], [641]])
def test_prompt_one_sequence(backend, lens):
    run_prompt(backend, lens, 2, 2, 128)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads,dim", [(3, 1, 64), (4, 1, 128), (2, 2, 96)])
def test_prompt_pages(backend, q_heads, kv_heads, dim, page):
    run_prompt(backend, [100, 1, 0, 37, 130], q_heads, kv_heads, dim, page, [0, 300, 64, 513, 41])


def test_prompt_queries_with_gaps(backend):
    run_prompt(backend, [70, 200], 4, 2, 64, q_apart=3)


def test_prompt_rows_without_keys(backend):
    """Fewer keys than rows: the first rows see nothing and are zeros."""
    import torch

    out = run_prompt(backend, [300, 5, 140], 2, 1, 64, 16, [-170, -5, -1])
    assert torch.count_nonzero(out[:170]) == 0 and torch.count_nonzero(out[300:305]) == 0 and torch.count_nonzero(out[305]) == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_prompt_unseen_keys_have_no_influence(backend, value):
    """Inf and NaN in keys and values reach the rows that see them and no others: rows before them, the next sequence, rows of a page behind the end."""

    def packed(q, keys, values, tables):
        values[60, 0, 5] = value
        keys[150, 1, 3] = value
        values[150, 1, 3] = value

    run_prompt(backend, [100, 129], 4, 2, 64, edit=packed)

    def paged(q, keys, values, tables):
        for x in (keys, values):
            x[int(tables[0][2]), :, 5:] = value  # 37 keys: rows 5 and on of the third page
            x[int(tables[1][8]), :, 2:] = value  # 130 keys

    run_prompt(backend, [37, 30], 4, 2, 128, 16, [0, 100], edit=paged)


def test_prompt_masks_of_the_lowest_value(backend):
    """Scores near the lowest fp32 and rows whose scores differ by more than fp32's exponents."""

    def edit(q, keys, values, tables):
        keys[:50] *= 1e18
        q[200:210] *= 1e18
        q[220] *= 1e-30

    run_prompt(backend, [256], 2, 1, 64, edit=edit)


def test_prompt_growing_maximum(backend):
    """The maximum grows from tile to tile, by little and by much."""

    def edit(q, keys, values, tables):
        import torch

        q[:] = q[:1]
        for t in range(0, keys.shape[0]):
            keys[t] = (q[0, :1] * (0.002 * t + (3 if t % 190 == 189 else 0))).to(torch.bfloat16)

    run_prompt(backend, [800], 1, 1, 128, edit=edit)


def tree_words(n, rng, shape):
    words = []
    for i in range(n):
        parent = i - 1 if shape == "chain" else int(rng.integers(max(0, i - 5), i)) if i else -1
        words.append((1 << i) | (words[parent] if i and shape != "none" else 0))
    if shape == "none":
        words = [0] * n
    return words


def run_tree(backend, lens, drafts, q_heads, kv_heads, dim, page, shape="tree", seed=0, edit=None, arrays=True, most=None):
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(seed)
    n = sum(drafts)
    q = normal(rng, n, q_heads, dim, scale=1.5)
    totals = [a + b for a, b in zip(lens, drafts)]
    tables, pages = pages_for(totals, page, rng)
    keys, values = normal(rng, pages, kv_heads, page, dim), normal(rng, pages, kv_heads, page, dim)
    words = [w for m in drafts for w in tree_words(m, rng, shape)]
    if edit:
        edit(q, keys, values, tables)
    out = torch.full((n, q_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    tab, ctx, off = torch.from_numpy(tables).cuda(), i32(lens), i32(offsets(drafts))
    anc = torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device="cuda")
    scale = 1 / math.sqrt(dim)
    torch.cuda.synchronize()
    op = A.TreeAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(tab), held(ctx), max_context=most or max(lens), max_drafts=max(drafts),
                         q_offsets=held(off) if arrays else None, ancestors=held(anc) if arrays else None, scale=scale)
    op.run()
    backend.synchronize_device()
    first = out.clone()
    for _ in range(2):  # the same bits every time
        out.fill_(7.0)
        torch.cuda.synchronize()
        op.run()
        backend.synchronize_device()
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))
    group, starts = q_heads // kv_heads, offsets(drafts)
    for s, (ctx_len, new) in enumerate(zip(lens, drafts)):
        total, rows = ctx_len + new, slice(starts[s], starts[s + 1])
        t = np.arange(total)
        where = torch.from_numpy(tables[s][t // page].astype(np.int64)).cuda()
        k, v = (x[where, :, torch.from_numpy(t % page).cuda()].double().cpu() for x in (keys, values))
        seen = torch.ones(new, total, dtype=torch.bool)
        for i in range(new):
            for j in range(new):
                seen[i, ctx_len + j] = bool(words[starts[s] + i] >> j & 1)
        heads = range(q_heads) if new * total * q_heads < 40000 else sorted({0, q_heads - 1, q_heads // 2})
        for h in heads:
            want, spread = formula(q[rows, h].double().cpu(), k[:, h // group], v[:, h // group], scale, seen)
            check(out[rows, h], want, spread)
    return out


@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 1), (12, 4), (40, 2)])
def test_tree_one_token(backend, q_heads, kv_heads, dim):
    run_tree(backend, [0, 1, 15, 16, 17, 130, 700], [1] * 7, q_heads, kv_heads, dim, 16)


@pytest.mark.parametrize("page", [16, 64, 128, 512])
@pytest.mark.parametrize("drafts", [[2, 1, 7], [16, 3, 1], [33, 64, 9], [1, 0, 5]])
def test_tree_drafts(backend, drafts, page):
    run_tree(backend, [37, 500, 0], drafts, 6, 2, 128, page)
    run_tree(backend, [1037, 20, 3], drafts, 4, 4, 64, page, shape="chain")


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(8, 1, 128), (16, 2, 64), (3, 1, 96), (64, 1, 128)])
@pytest.mark.parametrize("lens,drafts", [([3000, 700], [64, 40]), ([255, 128, 0, 1100], [9, 33, 17, 1]), ([129], [64])])
def test_tree_many_rows(backend, q_heads, kv_heads, dim, lens, drafts):
    """More rows than one tile, cut units and whole ones, key tiles that two groups share."""
    run_tree(backend, lens, drafts, q_heads, kv_heads, dim, 32)


def test_tree_many_rows_long_context(backend):
    run_tree(backend, [70001], [7], 8, 1, 128, 128)
    run_tree(backend, [9000, 8000], [20, 64], 4, 1, 64, 16)


def test_tree_many_units_of_many_rows(backend):
    rng = np.random.default_rng(15)
    run_tree(backend, [int(n) for n in rng.integers(0, 400, 60)], [int(n) for n in rng.integers(1, 65, 60)], 8, 2, 64, 16)


@pytest.mark.parametrize("drafts", [1, 12])
@pytest.mark.parametrize("seqs,longest", [(16, 1000), (20, 1400), (37, 900), (3, 1300)])
def test_tree_whole_and_cut_units(backend, drafts, seqs, longest):
    """About as many units as the device has SMs and more, alike and not, on both sides of the rule that cuts them."""
    run_tree(backend, [longest - 7 * i for i in range(seqs)], [drafts] * seqs, 32, 8, 64, 32)
    run_tree(backend, [longest] + [50] * (seqs - 1), [drafts] * seqs, 32, 8, 64, 32)


def test_tree_defaults(backend):
    """Without offsets and words: every sequence has max_drafts tokens, a chain."""
    run_tree(backend, [100, 333, 5], [4, 4, 4], 4, 2, 64, 16, shape="chain", arrays=False)


def test_tree_longer_bounds(backend):
    """Lengths lie on the device: the bounds of the call may be far above them."""
    run_tree(backend, [100, 33], [2, 3], 4, 2, 64, 16, most=1000)


def test_tree_many_sequences(backend):
    rng = np.random.default_rng(5)
    run_tree(backend, [int(n) for n in rng.integers(0, 90, 300)], [1 + int(n) for n in rng.integers(0, 3, 300)], 2, 1, 64, 16)


def test_tree_long_context(backend):
    run_tree(backend, [40013], [3], 8, 1, 128, 64)


def test_tree_rows_that_see_nothing(backend):
    import torch

    out = run_tree(backend, [0, 20], [3, 2], 4, 2, 64, 16, shape="none")
    assert torch.count_nonzero(out[:3]) == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_tree_unseen_keys_have_no_influence(backend, value):
    def edit(q, keys, values, tables):
        for x in (keys, values):
            x[int(tables[0][2]), :, 7:] = value  # 39 = 37 + 2 keys: behind the end
            x[int(tables[1][3]), 1, 4] = value   # position 52 of 50 + 9: the third draft, seen by some

    run_tree(backend, [37, 50], [2, 9], 4, 2, 64, 16, edit=edit)


# ------------------------------------------------------------------------------------------------ norms and rotation
def run_rope(backend, tokens, q_heads, kv_heads, dim, rot, dtype, norm, pairs, page, joined=False, gamma=True, offset=0, seed=0):
    """Outputs are bf16: off by at most 2^-8 of the exact value and the fp32 arithmetic's 2^-18 of the pair's magnitude (a dozen roundings of 2^-24 and the
    reciprocal root's 2^-22 on values up to 2 of the pair's)."""
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(seed)
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    wide = (q_heads + 2 * kv_heads) * dim + (3 if offset else 0)
    if joined:
        x = torch.from_numpy((rng.standard_normal((tokens, wide)) * 2).astype(np.float32)).to(kind).cuda()[:, offset:]
        q, k, v = (x[:, a * dim:b * dim].unflatten(1, (b - a, dim)) for a, b in ((0, q_heads), (q_heads, q_heads + kv_heads), (q_heads + kv_heads, q_heads + 2 * kv_heads)))
    else:
        q, k, v = (torch.from_numpy((rng.standard_normal((tokens, h, dim)) * 2).astype(np.float32)).to(kind).cuda() for h in (q_heads, kv_heads, kv_heads))
    gq, gk = (torch.from_numpy((1 + 0.3 * rng.standard_normal(dim)).astype(np.float32)).cuda() if norm and gamma else None for _ in range(2))
    table = torch.from_numpy(A.rope_table(tokens + 40, rot)).cuda() if rot else None
    pos = rng.integers(0, tokens + 40, tokens)
    positions = i32(pos)
    n_pages = -(-tokens // page) + 1 if page > 1 else tokens
    keys, values = (torch.full((n_pages, kv_heads, page, dim) if page > 1 else (tokens, kv_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slot = rng.permutation(n_pages * page)[:tokens].astype(np.int64) if page > 1 else np.arange(tokens)
    slots = torch.from_numpy(slot.copy()).cuda()
    if page > 1 and tokens > 2:
        slots[1] = -1
    q_out = torch.zeros(tokens, q_heads, dim, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    A.QkNormRope(backend.cuda_context, held(q), held(k), held(v), held(q_out), held(keys), held(values), held(positions), held(table), slots=held(slots) if page > 1 else None, norm=norm,
                 gamma_q=held(gq), gamma_k=held(gk), eps=1e-6, pairs=pairs).run()
    backend.synchronize_device()

    def turned(x, gamma):
        x = x.double().cpu()
        if norm:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 if gamma is None else gamma.double().cpu())
        y, size = x.clone(), x.abs()
        if rot:
            a = torch.arange(rot // 2) * (1 if pairs == "half" else 2)
            b = a + (rot // 2 if pairs == "half" else 1)
            c, s = (table.double().cpu()[torch.from_numpy(pos)][:, None, :, i] for i in (0, 1))
            y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
            size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
        return y, size

    def near(got, want, size):
        assert ((got.double().cpu() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-18 * size).all()

    near(q_out, *turned(q, gq))
    want, size = turned(k, gk)
    stored = [t for t in range(tokens) if int(slots[t]) >= 0]
    if page > 1:
        page_of, row = slots.cpu()[stored] // page, slots.cpu()[stored] % page
        got_k, got_v = keys.cpu()[page_of, :, row], values.cpu()[page_of, :, row]
        untouched = torch.ones(n_pages, page, dtype=torch.bool)
        untouched[page_of, row] = False
        assert (keys.cpu().transpose(1, 2)[untouched] == 7).all() and (values.cpu().transpose(1, 2)[untouched] == 7).all()
    else:
        got_k, got_v = keys.cpu(), values.cpu()
    near(got_k, want[stored], size[stored])
    assert torch.equal(got_v, v.cpu().bfloat16()[stored])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,rot", [(8, 8), (64, 64), (64, 16), (80, 40), (96, 64), (112, 56), (128, 128), (128, 0)])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
def test_rope(backend, dim, rot, pairs, dtype):
    run_rope(backend, 37, 5, 5, dim, rot, dtype, True, pairs, 16)
    run_rope(backend, 1, 12, 3, dim, rot, dtype, False, pairs, 32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset", [0, 1])
def test_rope_joined_rows(backend, dtype, offset):
    """q | k | v in one buffer; with an offset of one element nothing is aligned to more than that."""
    run_rope(backend, 19, 7, 1, 72, 64, dtype, True, "half", 1, joined=True, offset=offset)
    run_rope(backend, 300, 32, 8, 128, 128, dtype, True, "adjacent", 64, joined=True, offset=offset, gamma=False)


def test_rope_outside_the_table_or_the_cache(backend):
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    q, k, v = (torch.ones(4, 2, 64, device="cuda") for _ in range(3))
    keys, values = (torch.full((2, 2, 16, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out, table = torch.ones(4, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.from_numpy(A.rope_table(10, 64)).cuda()
    positions, slots = i32([0, 10, -1, 9]), torch.tensor([0, 1, 2, 32], dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    A.QkNormRope(backend.cuda_context, held(q), held(k), held(v), held(out), held(keys), held(values), held(positions), held(table), slots=held(slots)).run()
    with pytest.raises(N.WfError) as e:
        backend.synchronize_device()
    assert e.value.status == N.WF_ERR_INDEX
    assert torch.count_nonzero(out[1:]) == 0 and (out[0] == 1).all()
    stored = keys != 7
    assert stored[0, :, 0].all() and int(stored.sum()) == 128
    backend.synchronize_device()


# ------------------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("page,dim,heads", [(16, 8, 1), (64, 128, 3), (32, 72, 2), (256, 64, 1)])
def test_copy_pages(backend, page, dim, heads):
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(3)
    keys, values = normal(rng, 3, 9, heads, page, dim), normal(rng, 3, 9, heads, page, dim)
    want = [keys.clone(), values.clone()]
    pairs, rows = [(0, 7), (3, 1), (5, 6), (2, 2)], [page, 1, page // 2 + 1, 5]
    cache = A.KvCache(backend.cuda_context, 3, 9, page, heads, dim, keys=held(keys), values=held(values))
    d_pairs, d_rows = i32(pairs), i32(rows)
    torch.cuda.synchronize()
    cache.copy_pages(held(d_pairs), held(d_rows))
    backend.synchronize_device()
    for x in want:
        for (a, b), n in zip(pairs, rows):
            x[:, b, :, :n] = x[:, a, :, :n].clone()
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])
    cache.copy_pages(held(d_pairs[:1].contiguous()))
    backend.synchronize_device()
    assert torch.equal(keys[:, 7], keys[:, 0]) and torch.equal(values[:, 7], values[:, 0])
    cache.close()


@pytest.mark.parametrize("page,dim", [(16, 128), (64, 72)])
def test_compact(backend, page, dim):
    import torch

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(4)
    lens, drafts, layers, heads = [0, 14, 63, 200], 40, 2, 3
    tables, pages = pages_for([n + drafts for n in lens], page, rng)
    keys, values = normal(rng, layers, pages, heads, page, dim), normal(rng, layers, pages, heads, page, dim)
    kept = [sorted(rng.choice(drafts, n, replace=False).tolist()) for n in (30, 0, 1, 9)]
    kept[0][:3] = [0, 1, 2] if kept[0][3] > 2 else kept[0][:3]
    want = [keys.clone(), values.clone()]
    for x, src in zip(want, (keys, values)):
        for s, n in enumerate(lens):
            for i, j in enumerate(kept[s]):
                x[:, int(tables[s][(n + i) // page]), :, (n + i) % page] = src[:, int(tables[s][(n + j) // page]), :, (n + j) % page]
    cache = A.KvCache(backend.cuda_context, layers, pages, page, heads, dim, keys=held(keys), values=held(values))
    rows = np.full((4, drafts), -5, np.int32)
    for r, ids in zip(rows, kept):
        r[:len(ids)] = ids
    arrays = [torch.from_numpy(tables).cuda(), i32(lens), torch.from_numpy(rows).cuda(), i32([len(x) for x in kept])]
    torch.cuda.synchronize()
    cache.compact(*(held(x) for x in arrays))
    backend.synchronize_device()
    assert torch.equal(keys, want[0]) and torch.equal(values, want[1])
    cache.close()


def test_sequences_fork_and_end(backend):
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(6)
    keys, values = normal(rng, 2, 12, 2, 16, 64), normal(rng, 2, 12, 2, 16, 64)
    cache = A.KvCache(backend.cuda_context, 2, 12, 16, 2, 64, keys=held(keys), values=held(values))
    a = cache.sequence()
    slots = a.extend(37)
    assert a.pages == [0, 1, 2] and slots[0] == 0 and slots[36] == 36 and cache.free_pages() == 9
    torch.cuda.synchronize()
    b = a.fork()
    backend.synchronize_device()
    assert b.pages[:2] == a.pages[:2] and b.pages[2] == 3 and cache.holders(0) == 2 and cache.holders(2) == 1
    assert torch.equal(keys[:, 3, :, :5], keys[:, 2, :, :5]) and not torch.equal(keys[:, 3, :, 5], keys[:, 2, :, 5])
    assert b.extend(20)[0] == 3 * 16 + 5 and len(b.pages) == 4
    a.free()
    assert cache.free_pages() == 12 - 4 and cache.holders(0) == 1
    b.truncate(32)
    assert cache.free_pages() == 10
    with pytest.raises(N.WfError) as e:
        b.extend(16 * 11)
    assert e.value.status == N.WF_ERR_TOO_LARGE and b.tokens == 32 and cache.free_pages() == 10
    b.free()
    assert cache.free_pages() == 12
    cache.close()


# ------------------------------------------------------------------------------------------------ refusals, streams, recording
def test_pages_outside_the_cache(backend):
    """A page number outside the cache is not followed: its keys are not seen, the status says so, and other sequences are as they were."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(8)
    ctx, q = backend.cuda_context, normal(rng, 40, 2, 64)
    keys, values = normal(rng, 8, 1, 16, 64), normal(rng, 8, 1, 16, 64)
    for bad in (8, -1, 2**31 - 1):
        tables, out = i32([[0, bad, 2], [3, 4, 5]]), torch.zeros(40, 2, 64, dtype=torch.bfloat16, device="cuda")
        lens, off = i32([40, 40]), i32([0, 20, 40])
        torch.cuda.synchronize()
        A.PromptAttention(ctx, held(q), held(keys), held(values), held(out), held(off), tables=held(tables), k_lens=held(lens)).run()
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX
        seen = torch.arange(40)[None, :] <= torch.arange(20)[:, None] + 20
        seen[:, 16:32] = False
        flat = [x[[0, 1, 2]].transpose(1, 2).flatten(0, 1)[:40, 0].double().cpu() for x in (keys, values)]
        check(out[:20, 1], *formula(q[:20, 1].double().cpu(), flat[0], flat[1], 1 / 8, seen))
        other = [x[[3, 4, 5]].transpose(1, 2).flatten(0, 1)[:40, 0].double().cpu() for x in (keys, values)]
        check(out[20:, 1], *formula(q[20:, 1].double().cpu(), other[0], other[1], 1 / 8, torch.arange(40)[None, :] <= torch.arange(20)[:, None] + 20))
        context = i32([38, 38])
        small, four = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda"), q[:4].contiguous()
        torch.cuda.synchronize()
        A.TreeAttention(ctx, held(four), held(keys), held(values), held(small), held(tables), held(context), max_context=38, max_drafts=2).run()
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX
        seen2 = torch.arange(40)[None, :] <= torch.arange(2)[:, None] + 38
        check(small[2:, 0], *formula(four[2:, 0].double().cpu(), other[0], other[1], 1 / 8, seen2))
        seen2 = seen2.clone()
        seen2[:, 16:32] = False
        check(small[:2, 0], *formula(four[:2, 0].double().cpu(), flat[0], flat[1], 1 / 8, seen2))
        backend.synchronize_device()


def test_lengths_outside_their_range(backend):
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(9)
    ctx, q, out = backend.cuda_context, normal(rng, 8, 2, 64), torch.full((8, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    keys, values, tables = normal(rng, 8, 1, 16, 64), normal(rng, 8, 1, 16, 64), i32([[0, 1], [2, 3]])
    for lens in ([33, 20], [-1, 20]):  # two pages hold 32
        torch.cuda.synchronize()
        A.PromptAttention(ctx, held(q), held(keys), held(values), held(out), held(i32([0, 4, 8])), tables=held(tables), k_lens=held(i32(lens))).run()
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX and torch.count_nonzero(out[:4]) == 0
    for context in ([31, 20], [-3, 20], [26, 20]):  # with two new tokens; more than the call was told of
        out.fill_(7.0)
        torch.cuda.synchronize()
        A.TreeAttention(ctx, held(q[:4].contiguous()), held(keys), held(values), held(out[:4]), held(tables), held(i32(context)), max_context=25, max_drafts=2).run()
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX and torch.count_nonzero(out[:2]) == 0 and torch.count_nonzero(out[2:4]) > 0
    for off in ([0, 9], [4, 2], [-1, 4]):
        torch.cuda.synchronize()
        A.PromptAttention(ctx, held(q), held(normal(rng, 8, 1, 64)), held(normal(rng, 8, 1, 64)), held(out), held(i32(off))).run()
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX


def test_refusals(backend):
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    ctx, lib = backend.cuda_context, backend.cuda_context._lib
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    q, out, off, tab, one = bf(4, 4, 64), bf(4, 4, 64), i32([0, 4]), i32([[0]]), i32([4])

    def status(op):
        with pytest.raises(N.WfError) as e:
            op.run()
        return e.value.status

    pages = bf(2, 2, 16, 64)
    prompt = lambda **k: A.PromptAttention(ctx, held(q), held(k.pop("keys", pages)), held(k.pop("values", pages)), held(out), held(off), **k)  # noqa: E731
    assert status(prompt()) == N.WF_ERR_INVALID_ARGUMENT  # pages without tables
    assert status(prompt(keys=bf(4, 2, 64), values=bf(4, 2, 64), tables=held(tab), k_lens=held(one))) == N.WF_ERR_INVALID_ARGUMENT  # tables without pages
    assert status(prompt(keys=bf(4, 3, 64), values=bf(4, 3, 64))) == N.WF_ERR_SHAPE  # 4 heads over 3
    assert status(prompt(tables=held(tab), k_lens=held(one), scale=0.0)) == N.WF_ERR_INVALID_ARGUMENT
    assert status(prompt(tables=held(tab), k_lens=held(one), scale=float("nan"))) == N.WF_ERR_INVALID_ARGUMENT
    assert status(prompt(tables=held(tab), k_lens=held(one), layer=1)) == N.WF_ERR_SHAPE
    odd = bf(2, 2, 24, 64)
    assert status(prompt(keys=odd, values=odd, tables=held(tab), k_lens=held(one))) == N.WF_ERR_SHAPE
    with pytest.raises(ValueError):
        prompt(keys=bf(2, 2, 16, 72), values=bf(2, 2, 16, 72))  # another dimension than q's
    with pytest.raises(ValueError):
        prompt(keys=pages.float(), values=pages)
    big_q, big = bf(4, 4, 136), bf(4, 2, 136)
    assert status(A.PromptAttention(ctx, held(big_q), held(big), held(big), held(bf(4, 4, 136)), held(off))) == N.WF_ERR_SHAPE
    tree = lambda **k: A.TreeAttention(ctx, held(q), held(pages), held(pages), held(out), held(tab), held(one), max_context=4, **k)  # noqa: E731
    assert status(tree(max_drafts=65, q_offsets=held(off))) == N.WF_ERR_TOO_LARGE
    assert status(tree(max_drafts=3)) == N.WF_ERR_SHAPE  # 4 tokens are not 3 for one sequence
    x, table = torch.zeros(4, 2, 64, device="cuda"), torch.from_numpy(A.rope_table(8, 64)).cuda()
    rope = lambda **k: A.QkNormRope(ctx, held(x), held(x), held(x), held(bf(4, 2, 64)), held(bf(4, 2, 64)), held(bf(4, 2, 64)), k.pop("positions", held(one)), held(table), **k)  # noqa: E731
    with pytest.raises(ValueError):
        rope()  # one position for four tokens
    with pytest.raises(ValueError):
        rope(positions=held(i32([0, 1, 2, 3])), pairs="other")
    args = N.QkNormRopeArgs(tokens=1)
    cache = N.KvCacheArgs(pages.data_ptr(), pages.data_ptr(), 2, 1, 2, 16, 64)
    import ctypes

    assert lib.wf_qk_norm_rope(ctx.handle, ctypes.byref(args), ctypes.byref(cache), 0, 0) == N.WF_ERR_INVALID_ARGUMENT
    assert lib.wf_qk_norm_rope(ctx.handle, None, ctypes.byref(cache), 0, 0) == N.WF_ERR_INVALID_ARGUMENT
    assert lib.wf_prompt_attention(ctx.handle, ctypes.byref(N.PromptAttentionArgs(tokens=1, seqs=1)), None, 0, 0) == N.WF_ERR_INVALID_ARGUMENT
    assert lib.wf_tree_attention(ctx.handle, None, ctypes.byref(cache), 0, 0) == N.WF_ERR_INVALID_ARGUMENT
    assert lib.wf_cache_copy_pages(ctx.handle, ctypes.byref(cache), 0, 0, 1, 0) == N.WF_ERR_INVALID_ARGUMENT
    assert lib.wf_cache_compact(ctx.handle, ctypes.byref(cache), 0, 1, 0, 0, 1, 0, 1, 0) == N.WF_ERR_INVALID_ARGUMENT
    # nothing to do is not an error
    empty = i32([0])
    A.PromptAttention(ctx, held(bf(0, 4, 64)), held(bf(0, 2, 64)), held(bf(0, 2, 64)), held(bf(0, 4, 64)), held(empty)).run()
    backend.synchronize_device()


def test_other_stream_and_recording(backend):
    """A recorded step serves a growing cache: the lengths are read when it runs."""
    import torch

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    ctx = backend.cuda_context
    stream = ctx.create_stream()
    rng = np.random.default_rng(12)
    q, out = normal(rng, 2, 4, 64), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    keys, values, tables = normal(rng, 8, 2, 16, 64), normal(rng, 8, 2, 16, 64), i32([[0, 1, 2, 3], [4, 5, 6, 7]])
    context = i32([5, 9])
    op = A.TreeAttention(ctx, held(q), held(keys), held(values), held(out), held(tables), held(context), max_context=60)
    fill = A.PromptAttention(ctx, held(q), held(keys), held(values), held(out), held(i32([0, 1, 2])), tables=held(tables), k_lens=held(i32([6, 10])))
    torch.cuda.synchronize()
    ctx.graph_begin(stream)
    for call in (op, fill):
        with pytest.raises(N.WfError) as e:
            call.run(stream)  # its scratch is not there yet
        assert e.value.status == N.WF_ERR_RECORDING
    ctx.graph_destroy(ctx.graph_end(stream))
    op.run(stream)
    fill.run(stream)
    ctx.synchronize(stream)
    ctx.graph_begin(stream)
    op.run(stream)
    graph = ctx.graph_end(stream)
    for lens in ([5, 9], [6, 10], [59, 0]):
        context.copy_(torch.tensor(lens, dtype=torch.int32))
        out.zero_()
        torch.cuda.synchronize()
        ctx.graph_launch(graph, stream)
        ctx.synchronize(stream)
        for s, n in enumerate(lens):
            k, v = (x[4 * s:4 * s + 4].transpose(1, 2).flatten(0, 1)[:n + 1].double().cpu() for x in (keys, values))
            for h in range(4):
                check(out[s:s + 1, h], *formula(q[s:s + 1, h].double().cpu(), k[:, h // 2], v[:, h // 2], 1 / 8, torch.ones(1, n + 1, dtype=torch.bool)))
    ctx.graph_destroy(graph)
    ctx.destroy_stream(stream)
