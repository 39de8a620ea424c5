"""The decoder of generate.py: prompts, single tokens, trees of drafts and forks against the same model in 64 bits on the CPU.

Tolerance: projections of many tokens round activations and weights once to fp16 (2^-11), attention rounds q, k, v, its weights and its output to bf16 (2^-8);
through two layers the logits move by a few times 2^-8 of their size, measured on their largest.  That holds where scores are of the order of one, so
that 2^-8 of a score is a small part of a weight: the norms of q and k see to it, and where there are none the first norm's gamma is made a twentieth (with
synthetic weights of standard deviation 1.5, q and k then have about 1.2)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOLERANCE = 8 * 2.0**-8


def spec(**more):
    from warpforge_b200.generate import DecoderSpec
    from warpforge_b200.quant import QuantizationType

    return DecoderSpec(QuantizationType.Q8_0, 256, 4, 2, 64, 512, 2, 320, max_positions=512, **more)


@pytest.fixture(scope="module", params=[dict(qk_norm=False, pairs="adjacent"), dict(qk_norm=True, pairs="half")])
def model(request):
    from warpforge_b200.backend import CudaContext
    from warpforge_b200.generate import Decoder

    ctx = CudaContext(0)
    m = Decoder(ctx, spec(**request.param), pages=64, page_tokens=16, max_tokens=256)
    if not m.spec.qk_norm:
        for layer in range(m.spec.layers):
            name = f"gamma1_{layer}"
            m.host[name] = m.host[name] * np.float32(0.05)
            ctx.copy_to_device(m._const(name).ptr, m.host[name])
    m.exact = {}
    for layer, w in enumerate(m.weights):
        for n, x in w.items():
            m.exact[n, layer] = x.dequantize_to_array().astype(np.float64)
    m.exact["head"] = m.head.dequantize_to_array().astype(np.float64)
    yield m
    m.close()
    ctx.close()


def reference(m, tokens):
    """Logits of every token of one sequence."""
    s, host = m.spec, {k: v.astype(np.float64) for k, v in m.host.items()}
    n = len(tokens)

    def norm(x, g):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + s.eps) * g

    def turn(x):
        c, sn = host["rope"][:n, None, :, 0], host["rope"][:n, None, :, 1]
        half = s.head_dim // 2
        a, b = (slice(0, half), slice(half, None)) if s.pairs == "half" else (slice(0, None, 2), slice(1, None, 2))
        y = x.copy()
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * sn, x[..., b] * c + x[..., a] * sn
        return y

    h = host["embedding"][np.asarray(tokens)]
    for layer in range(s.layers):
        W = lambda name: m.exact[name, layer].T  # noqa: E731, B023
        x = norm(h, host[f"gamma1_{layer}"])
        q, k, v = ((x @ W(w)).reshape(n, -1, s.head_dim) for w in ("wq", "wk", "wv"))
        if s.qk_norm:
            q, k = norm(q, host[f"gamma_q_{layer}"]), norm(k, host[f"gamma_k_{layer}"])
        q, k = turn(q), turn(k)
        k, v = (np.repeat(x, s.q_heads // s.kv_heads, axis=1) for x in (k, v))
        scores = np.einsum("ihd,jhd->hij", q, k) / np.sqrt(s.head_dim)
        scores[:, np.triu(np.ones((n, n), bool), 1)] = -np.inf
        p = np.exp(scores - scores.max(-1, keepdims=True))
        att = np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), v).reshape(n, -1)
        h = h + att @ W("wo")
        x = norm(h, host[f"gamma2_{layer}"])
        g = x @ W("wgate")
        h = h + (g / (1 + np.exp(-g)) * (x @ W("wup"))) @ W("wdown")
    return norm(h, host["gamma"]) @ m.exact["head"].T


def near(got, want):
    assert np.max(np.abs(got - want)) <= TOLERANCE * np.max(np.abs(want))


def test_prompts_then_tokens(model):
    rng = np.random.default_rng(1)
    texts = [rng.integers(0, 320, n) for n in (100, 17, 1)]
    seqs = [model.sequence() for _ in texts]
    cut = [70, 17, 1]
    for got, t, c in zip(model.prefill(seqs, [t[:c] for t, c in zip(texts, cut)]), texts, cut):
        near(got, reference(model, t[:c]))
    for got, t in zip(model.prefill(seqs, [texts[0][70:], texts[1][:0], texts[2][:0]]), texts):  # the rest of one behind its past, nothing for the others
        near(got, reference(model, t)[len(t) - len(got):]) if len(got) else None
    more = [list(t) for t in texts]
    for _ in range(3):
        new = rng.integers(0, 320, 3)
        for t, x in zip(more, new):
            t.append(int(x))
        for got, t in zip(model.step(seqs, [[int(x)] for x in new]), more):
            near(got[0], reference(model, t)[-1])
    for s in seqs:
        s.free()
    assert model.cache.free_pages() == 64


def test_drafts_are_kept_and_forgotten(model):
    rng = np.random.default_rng(2)
    texts = [list(map(int, rng.integers(0, 320, n))) for n in (45, 90)]
    seqs = [model.sequence() for _ in texts]
    model.prefill(seqs, [np.array(t) for t in texts])
    #        0 - 1 - 3        0 - 2 - 4 - 5
    trees = [[-1, 0, 0, 1], [-1, -1, 0, 1, 2, 4]]
    drafts = [list(map(int, rng.integers(0, 320, len(t)))) for t in trees]
    for got, text, tree, draft in zip(model.step(seqs, drafts, trees), texts, trees, drafts):
        for i in range(len(tree)):
            path, j = [], i
            while j >= 0:
                path.insert(0, draft[j])
                j = tree[j]
            near(got[i], reference(model, text + path)[-1])
    kept = [[0, 1, 3], [0, 2, 4, 5]]
    model.keep(seqs, [len(d) for d in drafts], kept)
    texts = [t + [d[i] for i in k] for t, d, k in zip(texts, drafts, kept)]
    assert [s.tokens for s in seqs] == [len(t) for t in texts]
    fork = seqs[0].fork()
    for s, t in ((seqs, texts), ([fork], texts[:1])):
        new = [int(x) for x in rng.integers(0, 320, len(s))]
        for got, text, x in zip(model.step(s, [[x] for x in new]), t, new):
            near(got[0], reference(model, text + [x])[-1])
    for s in seqs + [fork]:
        s.free()
    assert model.cache.free_pages() == 64
