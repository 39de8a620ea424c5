"""NaN and Inf that a row does see, at every place of a tile (bounds and helpers as in test_gpu_attention.py)."""
import numpy as np
import pytest
from test_gpu_attention import backend, run_prompt, run_tree  # noqa: F401

pytestmark = pytest.mark.gpu

VALUES = [float("nan"), float("inf")]


def check_rows(out, q, bad, sees, value):
    """Head h of a sequence's rows (out, q [rows, heads, dim]) is NaN in the rows that see its bad key, which has the value in element bad[h][1], and no others: a
    score of NaN, or of plus infinity; with minus infinity the key has no weight.  sees: [rows, heads]."""
    import torch

    element = torch.tensor([e for _, e in bad], device="cuda")
    factor = q.float().gather(2, element[None, :, None].expand(q.shape[0], -1, 1))[..., 0]
    nan = sees & (factor > 0 if value == float("inf") else torch.ones_like(sees))
    assert torch.equal(torch.isnan(out).all(-1), nan) and torch.equal(torch.isnan(out).any(-1), nan)


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,rows,first", [(128, 201, 40), (128, 201, 0), (16, 300, 0), (16, 300, 16), (16, 300, 32), (16, 300, 48), (16, 300, 150), (16, 300, 171)])
def test_prompt_a_bad_key_reaches_the_rows_that_see_it(backend, heads, rows, first, dim, value):  # noqa: F811
    """Only the key is bad, its value is not; key first + h of head h.  128 heads: items of two tiles of rows; 16: of one, which two groups of warps share."""
    import torch

    bad, kept = [(first + h, h % dim) for h in range(heads)], {}

    def edit(q, keys, values, tables):
        for h, (t, e) in enumerate(bad):
            keys[t, h, e] = value
        kept["q"] = q

    out = run_prompt(backend, [rows, 3], heads, heads, dim, edit=edit)
    sees = torch.arange(rows, device="cuda")[:, None] >= torch.tensor([t for t, _ in bad], device="cuda")[None, :]
    check_rows(out[:rows], kept["q"][:rows], bad, sees, value)
    assert torch.isfinite(out[rows:]).all()


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page,first", [(16, 64), (256, 1220)])
def test_prompt_a_bad_key_of_the_past(backend, page, first, dim, value):  # noqa: F811
    import torch

    bad, kept = [(first + h, h % dim) for h in range(128)], {}

    def edit(q, keys, values, tables):
        for h, (t, e) in enumerate(bad):
            keys[int(tables[0][t // page]), h, t % page, e] = value
        kept["q"] = q

    out = run_prompt(backend, [30], 128, 128, dim, page, [1310], edit=edit)
    sees = torch.arange(1310, 1340, device="cuda")[:, None] >= torch.tensor([t for t, _ in bad], device="cuda")[None, :]
    check_rows(out, kept["q"], bad, sees, value)


def run_bad_tree(backend, contexts, drafts, q_heads, kv_heads, dim, page, place, value):  # noqa: F811
    """place(s, h): the position of kv head h's bad key in sequence s, or None.  Chains."""
    import torch

    kept = {}

    def edit(q, keys, values, tables):
        for s in range(len(contexts)):
            for h in range(kv_heads):
                t = place(s, h)
                if t is not None:
                    keys[int(tables[s][t // page]), h, t % page, h % dim] = value
        kept["q"] = q

    out = run_tree(backend, contexts, [drafts] * len(contexts), q_heads, kv_heads, dim, page, shape="chain", edit=edit)
    group = q_heads // kv_heads
    for s, context in enumerate(contexts):
        at = [place(s, h // group) for h in range(q_heads)]
        rows = slice(s * drafts, (s + 1) * drafts)
        sees = torch.arange(context, context + drafts, device="cuda")[:, None] >= torch.tensor([10**6 if t is None else t for t in at], device="cuda")[None, :]
        check_rows(out[rows], kept["q"][rows], [(0, h // group % dim) for h in range(q_heads)], sees, value)


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("drafts,context", [(40, 100), (12, 400), (1, 100)])
def test_tree_a_bad_key_reaches_the_rows_that_see_it(backend, drafts, context, dim, value):  # noqa: F811
    """Rows on the 5th-generation tensor cores (160 and 48 of a kv head) and on mma.sync (4); keys of the context and drafted ones."""
    run_bad_tree(backend, [context, context], drafts, 256, 64, dim, 16, lambda s, h: h + s * (context - 30) if h + s * (context - 30) < context + drafts else None, value)


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("drafts", [20, 1])
def test_tree_a_bad_key_of_a_cut_unit(backend, drafts, value):  # noqa: F811
    for first in range(0, 64, 8):
        run_bad_tree(backend, [6000], drafts, 32, 8, 64, 64, lambda s, h: first + h + (3000 + 7 * first if h % 2 else 0), value)  # noqa: B023


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("dim,rot", [(64, 16), (80, 40), (96, 64), (128, 64), (128, 8)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rope_an_element_that_is_not_rotated_stays_alone(backend, dim, rot, pairs, dtype, value):  # noqa: F811
    """Token t has NaN or Inf in element rot + t of q and k: the other elements are as they are without it."""
    import torch
    from test_gpu_attention import held, i32

    from warpforge_b200 import attention as A

    rng = np.random.default_rng(dim + rot)
    tokens = dim - rot
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    fine = [torch.from_numpy(rng.standard_normal((tokens, h, dim)).astype(np.float32)).to(kind).cuda() for h in (3, 2, 2)]
    table, positions, at = torch.from_numpy(A.rope_table(tokens, rot)).cuda(), i32(range(tokens)), torch.arange(tokens, device="cuda")

    def run(q, k, v):
        out, keys, values = (torch.zeros(tokens, h, dim, dtype=torch.bfloat16, device="cuda") for h in (3, 2, 2))
        torch.cuda.synchronize()
        A.QkNormRope(backend.cuda_context, held(q), held(k), held(v), held(out), held(keys), held(values), held(positions), held(table), pairs=pairs).run()
        backend.synchronize_device()
        return out, keys

    want = run(*fine)
    for x in fine[:2]:
        x[at, :, rot + at] = value
    for got, ref in zip(run(*fine), want):
        ref[at, :, rot + at] = value
        assert torch.equal(torch.nan_to_num(got.float(), 12345.0), torch.nan_to_num(ref.float(), 12345.0))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("drafts", [1, 3, 12])
def test_tree_bad_pages_in_short_units(backend, drafts, dim):  # noqa: F811
    """Many short sequences a CTA, every third of which names a page outside the cache: its keys are not seen, the status says so, the others are as they were."""
    import torch
    from test_gpu_attention import check, formula, held, i32, normal

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(drafts + dim)
    seqs, page, pages = 700, 16, 64
    contexts = [int(n) for n in rng.integers(0, 40, seqs)]
    tables = rng.integers(0, pages, (seqs, 4)).astype(np.int32)
    gone = {s: int(rng.integers(0, -(-(contexts[s] + drafts) // page))) for s in range(0, seqs, 3)}
    for s, i in gone.items():
        tables[s, i] = (pages, -1, 2**31 - 1)[s % 9 // 3]
    q, keys, values = normal(rng, seqs * drafts, 4, dim), normal(rng, pages, 1, page, dim), normal(rng, pages, 1, page, dim)
    out, tab, ctx = torch.zeros_like(q), torch.from_numpy(tables).cuda(), i32(contexts)
    torch.cuda.synchronize()
    op = A.TreeAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(tab), held(ctx), max_context=40, max_drafts=drafts)
    first = None
    for _ in range(10):
        op.run()
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX
        first = out.clone() if first is None else first
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))
    host = [x.double().cpu() for x in (q, keys, values)]
    for s in list(range(0, 60)) + list(range(660, 700)):
        total, rows = contexts[s] + drafts, slice(s * drafts, (s + 1) * drafts)
        t = np.arange(total)
        named = np.where((tables[s] < 0) | (tables[s] >= pages), 0, tables[s])[t // page]
        k, v = (x[named, 0, t % page] for x in host[1:])
        seen = torch.from_numpy((t[None, :] <= np.arange(drafts)[:, None] + contexts[s]) & (t[None, :] // page != gone.get(s, -1)))
        check(out[rows, 3], *formula(host[0][rows, 3], k, v, dim**-0.5, seen))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 5])
def test_prompt_bad_pages_beside_good_ones(backend, heads, dim):  # noqa: F811
    """The same for prompts: rows before the page that is not there, and other sequences, do not depend on when it is found."""
    import torch
    from test_gpu_attention import check, formula, held, i32, normal, offsets

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(heads + dim)
    seqs, page, pages = 150, 32, 40
    lens = [int(n) for n in rng.integers(1, 500 // heads, seqs)]
    tables = rng.integers(0, pages, (seqs, 16)).astype(np.int32)
    gone = {s: int(rng.integers(0, -(-lens[s] // page))) for s in range(0, seqs, 3)}
    for s, i in gone.items():
        tables[s, i] = (pages, -1, 2**31 - 1)[s % 9 // 3]
    n, starts = sum(lens), offsets(lens)
    q, keys, values = normal(rng, n, heads, dim), normal(rng, pages, 1, page, dim), normal(rng, pages, 1, page, dim)
    out, tab, off, k_lens = torch.zeros_like(q), torch.from_numpy(tables).cuda(), i32(starts), i32(lens)
    torch.cuda.synchronize()
    op = A.PromptAttention(backend.cuda_context, held(q), held(keys), held(values), held(out), held(off), tables=held(tab), k_lens=held(k_lens))
    first = None
    for _ in range(10):
        op.run()
        with pytest.raises(N.WfError) as e:
            backend.synchronize_device()
        assert e.value.status == N.WF_ERR_INDEX
        first = out.clone() if first is None else first
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))
    host = [x.double().cpu() for x in (q, keys, values)]
    for s in range(12):
        rows, t = slice(starts[s], starts[s + 1]), np.arange(lens[s])
        named = np.where((tables[s] < 0) | (tables[s] >= pages), 0, tables[s])[t // page]
        k, v = (x[named, 0, t % page] for x in host[1:])
        seen = torch.from_numpy((t[None, :] <= t[:, None]) & (t[None, :] // page != gone.get(s, -1)))
        check(out[rows, 0], *formula(host[0][rows, 0], k, v, dim**-0.5, seen))


def test_prompt_pasts_of_very_different_lengths(backend):  # noqa: F811
    """Some with none beside some with much, more sequences than a warp has lanes; two or one tile of rows an item."""
    rng = np.random.default_rng(21)
    for q_heads, seqs in ((8, 70), (64, 40), (128, 5)):
        past = [int(n) if i % 7 == 3 else 0 for i, n in enumerate(rng.integers(2000, 6000, seqs))]
        run_prompt(backend, [int(n) for n in rng.integers(0, 9, seqs)], q_heads, 1, 64, 64, past)


def test_prompt_time_does_not_grow_with_the_distance_of_pasts(backend):  # noqa: F811
    """One token behind 60,000 others, beside 40 short prompts, with 128 query heads for the kv head, so that an item has two tokens: 30,000 places between the
    first item and the others.  The token's 469 key tiles are one CTA's work, 1000 to 1700 cycles each with one or two groups of warps at them: below 1 ms, with the prompts
beside it or without; twice that is allowed."""
    import torch
    from test_gpu_attention import held, i32, normal, offsets

    from warpforge_b200 import attention as A

    rng, ctx, page = np.random.default_rng(22), backend.cuda_context, 64
    keys, values = normal(rng, 1024, 1, page, 64), normal(rng, 1024, 1, page, 64)
    start, stop = ctx.create_event(), ctx.create_event()

    def took(lens, past):
        q = normal(rng, sum(lens), 128, 64)
        out, tables = torch.zeros_like(q), torch.from_numpy(rng.integers(0, 1024, (len(lens), 1024)).astype(np.int32)).cuda()
        off, k_lens = i32(offsets(lens)), i32([a + b for a, b in zip(lens, past)])
        torch.cuda.synchronize()
        op = A.PromptAttention(ctx, held(q), held(keys), held(values), held(out), held(off), tables=held(tables), k_lens=held(k_lens))
        times = []
        for _ in range(5):
            ctx.record_event(start)
            op.run()
            ctx.record_event(stop)
            backend.synchronize_device()
            times.append(ctx.elapsed_ms(start, stop))
        return min(times)

    alone, both = took([1], [60000]), took([1] + [5] * 40, [60000] + [0] * 40)
    assert alone <= 2.0 and both <= 2.0, (alone, both)


def test_what_the_error_says(backend):  # noqa: F811
    """A page outside the cache is not reported as an embedding's index."""
    import torch
    from test_gpu_attention import held, i32, normal

    from warpforge_b200 import _native as N
    from warpforge_b200 import attention as A

    rng = np.random.default_rng(1)
    q, pages = normal(rng, 1, 1, 64), normal(rng, 2, 1, 16, 64)
    tables, context, out = i32([[2]]), i32([3]), torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    A.TreeAttention(backend.cuda_context, held(q), held(pages), held(pages), held(out), held(tables), held(context), max_context=3).run()
    with pytest.raises(N.WfError, match="a page") as e:
        backend.synchronize_device()
    assert e.value.status == N.WF_ERR_INDEX
