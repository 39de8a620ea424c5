"""Attention over packed prompts and over a paged cache against the formulas in 64 bits, at the sizes and masks where kernels go wrong.

Tolerances.  Outputs are bf16: a rounded result is off by at most 2^-9 of itself, 2^-8 between two neighbours.  The prompt kernel rounds the
weights to bf16 before the second product: each is off by at most 2^-9 of itself, so the sum by at most 2^-9 sum_t p_t |v_t|, which `spread`
below is (the largest over the elements of a row).  Scores come from exact products summed in fp32 (dim <= 128 terms: 128 * 2^-24 of the sum of their magnitudes,
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
