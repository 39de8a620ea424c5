"""Sequences of the decoder that share pages and then go separate ways, against the same model in 64 bits (tolerance as in test_gpu_generate.py)."""
import numpy as np
import pytest
from test_gpu_generate import model, near, reference  # noqa: F401

pytestmark = pytest.mark.gpu


def goes_on(model, rng, seqs, texts, tokens=3):  # noqa: F811
    """Some tokens more for each sequence, all of them in every step."""
    for _ in range(tokens):
        new = [int(x) for x in rng.integers(0, 320, len(seqs))]
        for got, text, x in zip(model.step(seqs, [[x] for x in new]), texts, new):
            text.append(x)
            near(got[0], reference(model, text)[-1])


def test_a_fork_is_cut_back_and_goes_on(model):  # noqa: F811
    rng = np.random.default_rng(11)
    text = list(map(int, rng.integers(0, 320, 45)))
    a = model.sequence()
    model.prefill([a], [np.array(text)])
    b, c = a.fork(), a.fork()
    for s, n in ((a, 20), (c, 33)):  # inside pages that all of them hold
        s.truncate(n)
    texts = [text[:20], list(text), text[:33]]
    more = rng.integers(0, 320, 9)
    near(model.prefill([a], [more])[0], reference(model, texts[0] + more.tolist())[20:])
    texts[0] += more.tolist()
    goes_on(model, rng, [a, b, c], texts)
    for s in (a, b, c):
        s.free()
    assert model.cache.free_pages() == 64


def test_a_fork_between_drafts_and_what_is_kept(model):  # noqa: F811
    """Two sequences keep different paths of the same drafts, which lie in pages that both hold."""
    rng = np.random.default_rng(12)
    for start in (10, 45):
        text = list(map(int, rng.integers(0, 320, start)))
        a = model.sequence()
        model.prefill([a], [np.array(text)])
        tree = [-1, 0, 0, 1, 2, 3, 4, 6, 7, 8, 9, 10, 5, 12] + [13 + i for i in range(12)]
        draft = list(map(int, rng.integers(0, 320, len(tree))))
        model.step([a], [draft], [tree])
        b = a.fork()

        def path(i):
            return [] if i < 0 else path(tree[i]) + [i]

        kept = [path(11), path(25)]
        model.keep([a], [len(tree)], kept[:1])
        model.keep([b], [len(tree)], kept[1:])
        texts = [text + [draft[i] for i in k] for k in kept]
        assert [a.tokens, b.tokens] == [len(t) for t in texts]
        goes_on(model, rng, [a, b], texts)
        for s in (a, b):
            s.free()
        assert model.cache.free_pages() == 64
