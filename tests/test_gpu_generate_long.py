"""The decoder with shared prefixes and with selected pages, from prompts over forks, single tokens, trees of drafts and what of them is kept, against the same model in 64 bits
on the CPU.  Tolerance as in test_gpu_generate.py, for the reasons given there.

A decoder that selects pages is held against a model that sees the keys of the pages which it says it has selected (its last call's lists are in its buffers), and the
lists against the definition, from the bounds that it holds and the queries that it used: both are exact."""
import numpy as np
import pytest

from test_gpu_generate import near, reference
from test_gpu_select import bounds_of, plain_list

pytestmark = pytest.mark.gpu


def make(layers=2, **more):
    from warpforge_b200.backend import CudaContext
    from warpforge_b200.generate import Decoder, DecoderSpec
    from warpforge_b200.quant import QuantizationType

    ctx = CudaContext(0)
    spec = DecoderSpec(QuantizationType.Q8_0, 256, 4, 2, 64, 512, layers, 320, max_positions=512, qk_norm=True, pairs="half")
    m = Decoder(ctx, spec, pages=80, page_tokens=16, max_tokens=400, **more)
    m.exact = {(n, layer): x.dequantize_to_array().astype(np.float64) for layer, w in enumerate(m.weights) for n, x in w.items()}
    m.exact["head"] = m.head.dequantize_to_array().astype(np.float64)
    return m


def closed(m):
    assert m.cache.free_pages() == 80
    m.close()
    m.ctx.close()


def paths(tree, draft):
    for i in range(len(tree)):
        path, j = [], i
        while j >= 0:
            path.insert(0, draft[j])
            j = tree[j]
        yield path


@pytest.mark.parametrize("more", [dict(share_prefixes=True), dict(selected_pages=64)])
def test_forks_drafts_and_tokens(more):
    """With room for all pages a selection leaves nothing out: both decoders are the model."""
    m = make(**more)
    rng = np.random.default_rng(2)
    texts = [list(map(int, rng.integers(0, 320, n))) for n in (150, 40)]
    seqs = [m.sequence() for _ in texts]
    for got, t in zip(m.prefill(seqs, [np.array(t) for t in texts]), texts):
        near(got, reference(m, t))
    seqs = [seqs[0], seqs[0].fork(), seqs[0].fork(), seqs[1], seqs[1].fork()]
    texts = [list(texts[i]) for i in (0, 0, 0, 1, 1)]
    for _ in range(2):
        new = [int(x) for x in rng.integers(0, 320, 5)]
        for t, x in zip(texts, new):
            t.append(x)
        for got, t in zip(m.step(seqs, [[x] for x in new]), texts):
            near(got[0], reference(m, t)[-1])
    trees = [[-1, 0, 0, 1], [-1, -1, 0, 1, 2, 4], [-1], [-1, 0], [-1, -1, -1]]
    drafts = [list(map(int, rng.integers(0, 320, len(t)))) for t in trees]
    for got, text, tree, draft in zip(m.step(seqs, drafts, trees), texts, trees, drafts):
        for g, path in zip(got, paths(tree, draft)):
            near(g, reference(m, text + path)[-1])
    kept = [[0, 1, 3], [0, 2, 4, 5], [], [0, 1], [2]]
    m.keep(seqs, [len(d) for d in drafts], kept)
    texts = [t + [d[i] for i in k] for t, d, k in zip(texts, drafts, kept)]
    seqs.append(seqs[1].fork())
    texts.append(list(texts[1]))
    order = [1, 5, 0, 2, 4, 3]
    seqs, texts = [seqs[i] for i in order], [texts[i] for i in order]
    new = [int(x) for x in rng.integers(0, 320, 6)]
    for got, t, x in zip(m.step(seqs, [[x] for x in new]), texts, new):
        near(got[0], reference(m, t + [x])[-1])
    for s in seqs:
        s.free()
    closed(m)


def check_bounds(m, seqs):
    """Of every full page of the sequences."""
    spec, c = m.spec, m.cache
    keys = np.empty((spec.layers, c.page_count, spec.kv_heads, c.page_tokens, spec.head_dim), np.uint16)
    codes, scales = np.empty((*keys.shape[:3], 2, spec.head_dim), np.int8), np.empty(keys.shape[:3], np.float32)
    for host, d in ((keys, c.keys), (codes, m.bounds.codes), (scales, m.bounds.scales)):
        m.ctx.copy_to_host(host, d.ptr)
    import torch

    keys = torch.from_numpy((keys.astype(np.uint32) << 16).view(np.float32))
    for s in seqs:
        for page in s.pages[:s.tokens // c.page_tokens]:
            for layer in range(spec.layers):
                for h in range(spec.kv_heads):
                    want = bounds_of(keys[layer, page, h])
                    assert np.array_equal(codes[layer, page, h], want[0]) and scales[layer, page, h] == want[1]
    return codes.astype(np.float64), scales.astype(np.float64)


def test_few_pages_of_many():
    width, recent = 6, 16
    m = make(1, selected_pages=width, first_pages=1, recent_tokens=recent)
    spec, size = m.spec, m.cache.page_tokens
    rng = np.random.default_rng(3)
    texts = [list(map(int, rng.integers(0, 320, n))) for n in (200, 37, 121)]
    seqs = [m.sequence() for _ in texts]
    m.prefill(seqs, [np.array(t) for t in texts])
    seqs, texts = seqs + [seqs[0].fork()], texts + [list(texts[0])]
    for trees in ([[-1]] * 4, [[-1, 0, 0, 1], [-1], [-1, -1, 1], [-1]], [[-1]] * 4):
        drafts = [list(map(int, rng.integers(0, 320, len(t)))) for t in trees]
        context = [s.tokens for s in seqs]
        got = m.step(seqs, drafts, trees)
        n = sum(len(d) for d in drafts)
        lists, lens = np.empty((n, spec.kv_heads, width), np.int32), np.empty((n, spec.kv_heads, 2), np.int32)
        q = np.empty((n, spec.q_heads, spec.head_dim), np.uint16)
        for host, name in ((lists, "lists"), (lens, "list_lens"), (q, "qb")):
            m.ctx.copy_to_host(host, m.buf[name])
        q = (q.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        codes, scales = check_bounds(m, seqs)
        row = 0
        for s, text, tree, draft, c, g in zip(seqs, texts, trees, drafts, context, got):
            for i, path in enumerate(paths(tree, draft)):
                for h in range(spec.kv_heads):
                    want = plain_list(q[row, 2 * h:2 * h + 2], codes[0, :, h], scales[0, :, h], s.pages, c, len(tree), i, True, size, width, 1, recent)
                    assert (lists[row, h].tolist(), lens[row, h].tolist()) == want
                # the same token in a model that sees the keys of the listed pages
                seen = np.ones((spec.q_heads, c + len(path)), bool)
                for h in range(spec.q_heads):
                    there = set(lists[row, h // 2].tolist())
                    seen[h, :c] = [s.pages[t // size] in there for t in range(c)]
                assert seen.all() or c > (width - 2) * size
                near(g[i], masked(m, text + path, seen))
                row += 1
        kept = [list(range(len(t))) if all(p == i - 1 for i, p in enumerate(t)) else [0] for t in trees]
        m.keep(seqs, [len(d) for d in drafts], kept)
        texts = [t + [d[i] for i in k] for t, d, k in zip(texts, drafts, kept)]
        check_bounds(m, seqs)
    for s in seqs:
        s.free()
    closed(m)


def masked(m, tokens, seen):
    """Logits of the last token, which sees those keys (seen [q_heads, tokens]); one layer, so that its keys depend on nobody's attention."""
    s, host = m.spec, {k: v.astype(np.float64) for k, v in m.host.items()}
    n = len(tokens)
    W = lambda name: m.exact[name, 0].T  # noqa: E731

    def norm(x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + s.eps) * g

    def turn(x):
        c, sn = host["rope"][:n, None, :, 0], host["rope"][:n, None, :, 1]
        half = s.head_dim // 2
        a, b = x[..., :half], x[..., half:]
        return np.concatenate((a * c - b * sn, b * c + a * sn), -1)

    h = host["embedding"][np.asarray(tokens)]
    x = norm(h, host["gamma1_0"])
    q, k, v = ((x @ W(w)).reshape(n, -1, s.head_dim) for w in ("wq", "wk", "wv"))
    q, k = turn(norm(q, host["gamma_q_0"])), turn(norm(k, host["gamma_k_0"]))
    k, v = (np.repeat(x, s.q_heads // s.kv_heads, axis=1) for x in (k, v))
    scores = np.einsum("hd,jhd->hj", q[-1], k) / np.sqrt(s.head_dim)
    scores[~seen] = -np.inf
    p = np.exp(scores - scores.max(-1, keepdims=True))
    att = np.einsum("hj,jhd->hd", p / p.sum(-1, keepdims=True), v).reshape(-1)
    h = h[-1] + att @ W("wo")
    x = norm(h, host["gamma2_0"])
    g = x @ W("wgate")
    h = h + (g / (1 + np.exp(-g)) * (x @ W("wup"))) @ W("wdown")
    return norm(h, host["gamma"]) @ m.exact["head"].T
