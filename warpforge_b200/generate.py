"""A decoder of quantized projections and attention over a paged cache, from prompt to tokens.

    h += Wo . attention(rotated q, k; v)      q, k, v = W{q,k,v} . rms_norm(h)
    h += Wdown . (silu(gate) * up)            gate, up = W{gate,up} . rms_norm(h)
    logits = Whead . rms_norm(h)

Prompts of several sequences go through together (``prefill``: tensor-core GEMMs and PromptAttention), new tokens by ``step``: one for each sequence, or a
tree of drafted ones of which ``keep`` retains a path (decode GEMVs, TreeAttention, compaction of the cache).  New tokens may read the prefix that neighbouring
sequences share (forks) once for all of them (``share_prefixes``), or a few pages of a long context that promise the largest scores (``selected_pages``).  ``python -m
warpforge_b200.generate`` runs it on seeded synthetic weights and prints tokens per second.
"""
from __future__ import annotations

import argparse
import time
from contextlib import contextmanager
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence as Seq

import numpy as np

from . import _native as N
from . import attention as A
from . import quant as Q
from .backend import CudaContext, DeviceTensor, QuantizedWeight

SIZES = {"f32": 4, "bf16": 2, "i32": 4, "i64": 8}
MAX_DRAFTS = 64  # of a sequence in a step: an ancestors word's bits


@dataclass(frozen=True)
class DecoderSpec:
    qtype: Q.QuantizationType
    d_model: int
    q_heads: int
    kv_heads: int
    head_dim: int
    ffn: int
    layers: int
    vocab: int
    qk_norm: bool = False
    pairs: str = "adjacent"  # GGUF files of this model family hold q and k for pairs (2i, 2i + 1)
    rope_base: float = 10000.0
    max_positions: int = 4096
    eps: float = 1e-5

    def projections(self) -> Dict[str, tuple]:
        q, kv = self.q_heads * self.head_dim, self.kv_heads * self.head_dim
        return {"wq": (q, self.d_model), "wk": (kv, self.d_model), "wv": (kv, self.d_model), "wo": (self.d_model, q), "wgate": (self.ffn, self.d_model),
                "wup": (self.ffn, self.d_model), "wdown": (self.d_model, self.ffn)}


class Decoder:
    """Seeded synthetic weights; `max_tokens` rows of activations, a cache of `pages` pages.  A call that is refused or fails leaves the sequences as long
    as they were.

    share_prefixes: ``step`` reads what neighbours among its sequences have in common once for all of them.  selected_pages: in ``step`` a new token reads, for every kv head, so many pages
    at most: the first `first_pages`, those of the last `recent_tokens` tokens, those of the new ones, and the ones between whose bounds promise the largest scores (0: all pages)."""

    def __init__(self, context: CudaContext, spec: DecoderSpec, pages: int, page_tokens: int = 64, max_tokens: int = 512, max_sequences: int = 16, seed: int = 1,
                 share_prefixes: bool = False, selected_pages: int = 0, first_pages: int = 1, recent_tokens: int = 64):
        if selected_pages < 0 or first_pages < 0 or recent_tokens < 0 or (selected_pages and share_prefixes):
            raise ValueError(f"selected_pages {selected_pages}, first_pages {first_pages}, recent_tokens {recent_tokens}; not together with share_prefixes")
        self.ctx, self.spec, self.max_tokens, self.max_sequences = context, spec, max_tokens, max_sequences
        self.share_prefixes, self.selected_pages, self.first_pages, self.recent_tokens = share_prefixes, selected_pages, first_pages, recent_tokens
        if selected_pages:
            self._fits_lists(1, page_tokens)
        self.cache = A.KvCache(context, spec.layers, pages, page_tokens, spec.kv_heads, spec.head_dim)
        rng = np.random.default_rng(seed)
        self.host: Dict[str, np.ndarray] = {}
        self._owned: List[int] = []
        self._table_width = -(-spec.max_positions // page_tokens)

        def weight(rows, k, n):
            return QuantizedWeight(context, spec.qtype, Q.synth_weight(spec.qtype, rows, k, seed * 1000 + n), rows, k)

        self.weights = [{name: weight(r, k, 10 * layer + i) for i, (name, (r, k)) in enumerate(spec.projections().items())} for layer in range(spec.layers)]
        self.head = weight(spec.vocab, spec.d_model, 9999)
        gamma = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
        for layer in range(spec.layers):
            self._keep(f"gamma1_{layer}", gamma(spec.d_model))
            self._keep(f"gamma2_{layer}", gamma(spec.d_model))
            if spec.qk_norm:
                self._keep(f"gamma_q_{layer}", gamma(spec.head_dim))
                self._keep(f"gamma_k_{layer}", gamma(spec.head_dim))
        self._keep("gamma", gamma(spec.d_model))
        self._keep("embedding", rng.standard_normal((spec.vocab, spec.d_model)).astype(np.float32))
        self._keep("rope", A.rope_table(spec.max_positions, spec.head_dim, spec.rope_base))
        s = spec
        widths = {"h": s.d_model, "x": s.d_model, "t": s.d_model, "q": s.q_heads * s.head_dim, "k": s.kv_heads * s.head_dim, "v": s.kv_heads * s.head_dim, "gate": s.ffn,
                  "up": s.ffn, "act": s.ffn, "logits": s.vocab}
        self.buf = {n: self._alloc(max_tokens * w * 4) for n, w in widths.items()}
        self.buf["qb"], self.buf["att"] = (self._alloc(max_tokens * s.q_heads * s.head_dim * 2) for _ in range(2))
        # what a call says about its tokens and sequences
        self._room = {n: max_tokens * size for n, size in (("ids", 8), ("positions", 4), ("slots", 8), ("ancestors", 8))}
        self._room.update({n: (max_sequences + 1) * 4 for n in ("offsets", "lens", "counts")}, tables=max_sequences * self._table_width * 4, kept=max_sequences * MAX_DRAFTS * 4)
        if share_prefixes:
            self._room.update(groups=(max_sequences + 1) * 4, prefixes=(max_sequences + 1) * 4)
        self.bounds = A.PageBounds(self.cache) if selected_pages else None
        if selected_pages:
            self._room.update(before=(max_sequences + 1) * 4, moved=(max_sequences + 1) * 4)
            new = min(max_tokens, max_sequences * MAX_DRAFTS) * s.kv_heads  # lists of a step
            self._room.update(lists=new * selected_pages * 4, list_lens=new * 8)
        self._room = {n: max(room, 16) for n, room in self._room.items()}
        self.buf.update({n: self._alloc(room) for n, room in self._room.items()})

    def _alloc(self, nbytes: int) -> int:
        self._owned.append(self.ctx.allocate(max(nbytes, 16)))
        return self._owned[-1]

    def _keep(self, name: str, a: np.ndarray) -> None:
        self.host[name] = a
        setattr(self, "_" + name, DeviceTensor(self._alloc(a.nbytes), a.shape, "f32"))
        self.ctx.copy_to_device(getattr(self, "_" + name).ptr, a)

    def _const(self, name: str) -> DeviceTensor:
        return getattr(self, "_" + name)

    def _send(self, name: str, a, dtype: str) -> DeviceTensor:
        a = np.ascontiguousarray(a, {"i32": np.int32, "i64": np.int64}[dtype])
        if a.nbytes > self._room[name]:
            raise ValueError(f"{name}: {a.nbytes} bytes, room for {self._room[name]}")
        if a.size:
            self.ctx.copy_to_device(self.buf[name], a)
        return DeviceTensor(self.buf[name], a.shape, dtype)

    def sequence(self) -> A.Sequence:
        return self.cache.sequence()

    # ---- what a call may be, before any of it has happened; what it leaves where it fails later
    def _admit(self, sequences: Seq[A.Sequence], lens: Seq[int], positions: Seq[np.ndarray]) -> None:
        if len(sequences) != len(lens) or len({id(s) for s in sequences}) != len(sequences):
            raise ValueError(f"{len(lens)} entries for {len(sequences)} sequences, each of which is to be named once")
        if len(sequences) > self.max_sequences:
            raise ValueError(f"{len(sequences)} sequences, room for {self.max_sequences}")
        if sum(lens) > self.max_tokens:
            raise ValueError(f"{sum(lens)} tokens, room for {self.max_tokens}")
        for s, n, at in zip(sequences, lens, positions):
            if n and int(np.max(at)) >= self.spec.max_positions:
                raise ValueError(f"position {int(np.max(at))} of {self.spec.max_positions}")
            if s.tokens + n > self._table_width * self.cache.page_tokens:
                raise ValueError(f"a sequence of {s.tokens + n} tokens in tables for {self._table_width * self.cache.page_tokens}")

    @contextmanager
    def _extended(self, sequences: Seq[A.Sequence], lens: Seq[int]):
        """The slots of so many new tokens of each sequence; an exception inside makes the sequences as long as they were."""
        before = [s.tokens for s in sequences]
        try:
            yield np.concatenate([np.array(s.extend(n), np.int64) for s, n in zip(sequences, lens)])
        except BaseException:
            for s, n in zip(sequences, before):
                s.truncate(n)
            raise

    # ---- pages that are selected
    def _fits_lists(self, drafts: int, page_tokens: int) -> None:
        need = self.first_pages + (self.recent_tokens + drafts + page_tokens - 2) // page_tokens + 1
        if self.selected_pages < need:
            raise ValueError(f"{drafts} new tokens of a sequence need {need} pages in any case, {self.selected_pages} are selected")

    def _bound(self, tables: DeviceTensor, first: DeviceTensor, stop: DeviceTensor, most: int) -> None:
        """The bounds of the pages that new tokens went to, in all layers."""
        if self.bounds and most:
            self.bounds.update(tables, first, stop, max_tokens=most)

    # ---- the layers: `attend(layer, q, keys, values, out)` is the attention of this call
    def _layers(self, ids: np.ndarray, positions: np.ndarray, slots: np.ndarray, attend) -> None:
        ctx, lib, s, b, h = self.ctx, self.ctx._lib, self.spec, self.buf, self.ctx.handle
        n = len(ids)
        tokens = self._send("ids", ids, "i64")
        pos, slot = self._send("positions", positions, "i32"), self._send("slots", slots, "i64")
        part = lambda name, heads, dtype: DeviceTensor(b[name], (n, heads, s.head_dim), dtype)  # noqa: E731

        def linear(w, x, y, dtype=N.WF_DTYPE_F32):
            ctx._ck("wf_qlinear", lib.wf_qlinear(h, w.handle, x, dtype, 1, n, y, 1, 0))

        def norm(gamma):
            ctx._ck("wf_rms_norm", lib.wf_rms_norm(h, b["h"], gamma.ptr, b["x"], n, s.d_model, s.eps, 0))

        ctx._ck("wf_embedding", lib.wf_embedding(h, tokens.ptr, self._const("embedding").ptr, b["h"], n, s.vocab, s.d_model, 0))
        for layer, w in enumerate(self.weights):
            norm(self._const(f"gamma1_{layer}"))
            for name in ("q", "k", "v"):
                linear(w["w" + name], b["x"], b[name])
            keys, values = self.cache.layer(layer)
            gammas = {g: self._const(f"{g}_{layer}") for g in ("gamma_q", "gamma_k")} if s.qk_norm else {}
            A.QkNormRope(ctx, part("q", s.q_heads, "f32"), part("k", s.kv_heads, "f32"), part("v", s.kv_heads, "f32"), part("qb", s.q_heads, "bf16"), keys, values, pos,
                         self._const("rope"), slots=slot, norm=s.qk_norm, eps=s.eps, pairs=s.pairs, **gammas).run()
            attend(layer, part("qb", s.q_heads, "bf16"), keys, values, part("att", s.q_heads, "bf16"))
            linear(w["wo"], b["att"], b["t"], N.WF_DTYPE_BF16)
            ctx._ck("wf_add", lib.wf_add(h, b["h"], b["t"], b["h"], n * s.d_model, 0))
            norm(self._const(f"gamma2_{layer}"))
            linear(w["wgate"], b["x"], b["gate"])
            linear(w["wup"], b["x"], b["up"])
            ctx._ck("wf_swiglu", lib.wf_swiglu(h, b["gate"], b["up"], b["act"], n * s.ffn, 0))
            linear(w["wdown"], b["act"], b["t"])
            ctx._ck("wf_add", lib.wf_add(h, b["h"], b["t"], b["h"], n * s.d_model, 0))
        norm(self._const("gamma"))
        linear(self.head, b["x"], b["logits"])

    def _logits(self, n: int) -> np.ndarray:
        out = np.empty((n, self.spec.vocab), np.float32)
        if n:
            self.ctx.copy_to_host(out, self.buf["logits"])
        self.ctx.synchronize()  # reports what the kernels found
        return out

    def _tables(self, sequences: Seq[A.Sequence]) -> DeviceTensor:
        return self._send("tables", self.cache.tables(sequences, self._table_width), "i32")

    def prefill(self, sequences: Seq[A.Sequence], prompts: Seq[np.ndarray]) -> List[np.ndarray]:
        """The prompts behind what the sequences hold already; logits [len(prompt), vocab] of each."""
        lens = [len(p) for p in prompts]
        positions = [s.tokens + np.arange(n) for s, n in zip(sequences, lens)]
        self._admit(sequences, lens, positions)
        offsets = np.concatenate(([0], np.cumsum(lens)))
        with self._extended(sequences, lens) as slots:
            tables, off = self._tables(sequences), self._send("offsets", offsets, "i32")
            total = self._send("lens", [s.tokens for s in sequences], "i32")
            self._layers(np.concatenate(prompts), np.concatenate(positions), slots,
                         lambda layer, q, k, v, out: A.PromptAttention(self.ctx, q, k, v, out, off, tables=tables, k_lens=total).run())
            if self.bounds:
                self._bound(tables, self._send("before", [s.tokens - n for s, n in zip(sequences, lens)], "i32"), total, max(lens, default=0))
            logits = self._logits(int(offsets[-1]))
        return [logits[a:b] for a, b in zip(offsets, offsets[1:])]

    def step(self, sequences: Seq[A.Sequence], tokens: Seq[Seq[int]], parents: Optional[Seq[Seq[int]]] = None) -> List[np.ndarray]:
        """New tokens of each sequence (one, or up to 64 drafted ones): parents[s][i] is the index of token i's parent among them, -1: the
        context; not given: a chain.  Logits [len(tokens[s]), vocab]; the tokens stay in the cache until ``keep`` says which of them remain."""
        lens = [len(t) for t in tokens]
        if max(lens, default=0) > MAX_DRAFTS:
            raise ValueError(f"{max(lens)} new tokens of a sequence, at most {MAX_DRAFTS}")
        if self.selected_pages and any(lens):
            self._fits_lists(max(lens), self.cache.page_tokens)
        context = [s.tokens for s in sequences]
        words, depth = [], []
        for s, n in enumerate(lens):
            seen = []
            for i in range(n):
                parent = i - 1 if parents is None else parents[s][i]
                if not -1 <= parent < i:
                    raise ValueError(f"token {i} with parent {parent}")
                seen.append((seen[parent][0] | (1 << i), seen[parent][1] + 1) if parent >= 0 else (1 << i, 0))
            words += [w for w, _ in seen]
            depth.append(np.array([d for _, d in seen], np.int64))
        positions = [c + d for c, d in zip(context, depth)]
        self._admit(sequences, lens, positions)
        offsets = np.concatenate(([0], np.cumsum(lens)))
        with self._extended(sequences, lens) as slots:
            tables, off, ctx_lens = self._tables(sequences), self._send("offsets", offsets, "i32"), self._send("lens", context, "i32")
            anc = self._send("ancestors", np.array(words, np.uint64).view(np.int64), "i64")
            self._layers(np.concatenate([np.asarray(t) for t in tokens]), np.concatenate(positions), slots, self._attention(sequences, context, lens, tables, off, ctx_lens, anc))
            if self.bounds:
                self._bound(tables, ctx_lens, self._send("before", [s.tokens for s in sequences], "i32"), max(lens, default=0))
            logits = self._logits(int(offsets[-1]))
        return [logits[a:b] for a, b in zip(offsets, offsets[1:])]

    def _attention(self, sequences: Seq[A.Sequence], context: List[int], lens: List[int], tables: DeviceTensor, off: DeviceTensor, ctx_lens: DeviceTensor, anc: DeviceTensor):
        """What a step's new tokens do in every layer: attend to all that their sequences hold, with a common prefix read once, or to selected pages."""
        ctx, drafts = self.ctx, dict(q_offsets=off, max_drafts=max(lens, default=1))
        if self.selected_pages:
            n = sum(lens)
            lists = DeviceTensor(self.buf["lists"], (n, self.spec.kv_heads, self.selected_pages), "i32")
            list_lens = DeviceTensor(self.buf["list_lens"], (n, self.spec.kv_heads, 2), "i32")

            def selected(layer, q, k, v, out):
                A.SelectPages(ctx, q, *self.bounds.layer(layer), tables, ctx_lens, lists, list_lens, page_tokens=self.cache.page_tokens, max_context=max(context, default=0), first=self.first_pages,
                              recent=self.recent_tokens, tree=True, **drafts).run()
                A.SelectedAttention(ctx, q, k, v, out, lists, list_lens, ancestors=anc).run()

            return selected
        if self.share_prefixes and sequences:
            groups, prefix = self.cache.shared_prefixes(sequences, context)
            if prefix.any():
                d_groups, d_prefix = self._send("groups", groups, "i32"), self._send("prefixes", prefix, "i32")
                own = max(c - int(p) for c, p in zip(context, np.repeat(prefix, np.diff(groups))))
                return lambda layer, q, k, v, out: A.SharedPrefixAttention(ctx, q, k, v, out, tables, ctx_lens, d_groups, d_prefix, max_prefix=int(prefix.max()), max_own=own, ancestors=anc,
                                                                           **drafts).run()
        return lambda layer, q, k, v, out: A.TreeAttention(ctx, q, k, v, out, tables, ctx_lens, max_context=max(context), ancestors=anc, **drafts).run()

    def keep(self, sequences: Seq[A.Sequence], drafted: Seq[int], kept: Seq[Seq[int]]) -> None:
        """After ``step`` with drafted[s] tokens: those of kept[s] (ascending, a path of the tree) remain, moved up to the end of the context."""
        if not len(sequences) == len(drafted) == len(kept) or len({id(s) for s in sequences}) != len(sequences):
            raise ValueError(f"{len(drafted)} and {len(kept)} entries for {len(sequences)} sequences, each of which is to be named once")
        for s, n, k in zip(sequences, drafted, kept):
            if not 0 <= n <= s.tokens or any(not before < i < n for before, i in zip([-1, *k], k)):
                raise ValueError(f"tokens {list(k)} of {n} drafted ones in a sequence of {s.tokens}")
        width = max([1] + [len(k) for k in kept])
        rows = np.zeros((len(sequences), width), np.int32)
        for row, k in zip(rows, kept):
            row[:len(k)] = k
        context = [s.tokens - n for s, n in zip(sequences, drafted)]
        still = [next((i for i, j in enumerate(k) if i != j), len(k)) for k in kept]  # tokens that lie where they belong
        moved = [(c + n, c + len(k)) for c, n, k in zip(context, still, kept)]
        self.cache.own(sequences, moved)
        tables, lens = self._tables(sequences), self._send("lens", context, "i32")
        self.cache.compact(tables, lens, self._send("kept", rows, "i32"), self._send("counts", [len(k) for k in kept], "i32"))
        if self.bounds:  # of the pages that tokens moved to.  Where none did, others may hold more of a page than is kept here, and ``step`` has left the bounds of all of it
            self._bound(tables, self._send("moved", [a for a, _ in moved], "i32"), self._send("before", [b for _, b in moved], "i32"), max((b - a for a, b in moved), default=0))
        self.ctx.synchronize()
        for s, c, k in zip(sequences, context, kept):
            s.truncate(c + len(k))

    def close(self) -> None:
        for w in [w for layer in self.weights for w in layer.values()] + [self.head]:
            w.close()
        for p in self._owned:
            self.ctx.free(p)
        self._owned = []
        if self.bounds:
            self.bounds.close()
        self.cache.close()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--qtype", default="Q4_0")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--d-model", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--ffn", type=int, default=11008)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--samples", type=int, default=1, help="continuations of each prompt, which share its pages")
    ap.add_argument("--share-prefixes", action="store_true", help="read what they share once for all of them")
    ap.add_argument("--selected-pages", type=int, default=0, help="pages that a new token reads (0: all)")
    a = ap.parse_args()
    spec = DecoderSpec(Q.QuantizationType[a.qtype], a.d_model, a.heads, a.kv_heads, a.d_model // a.heads, a.ffn, a.layers, a.vocab)
    ctx = CudaContext(0)
    need = a.sequences * a.samples * (-(-(a.prompt + a.tokens) // 64) + 1)
    model = Decoder(ctx, spec, pages=need, max_tokens=a.sequences * max(a.prompt, a.samples), max_sequences=a.sequences * a.samples, share_prefixes=a.share_prefixes,
                    selected_pages=a.selected_pages)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, a.vocab, a.prompt) for _ in range(a.sequences)]
    samples = lambda seqs: [s if i == 0 else s.fork() for s in seqs for i in range(a.samples)]  # noqa: E731
    warm = [model.sequence() for _ in prompts]
    model.prefill(warm, prompts)
    warm = samples(warm)
    if a.tokens > 1:  # else nothing is decoded, and a prompt may have every position that there is
        model.step(warm, [[0]] * len(warm))
    for s in warm:
        s.free()
    seqs = [model.sequence() for _ in prompts]
    t0 = time.perf_counter()
    last = [int(np.argmax(x[-1])) for x in model.prefill(seqs, prompts)]
    t1 = time.perf_counter()
    seqs = samples(seqs)
    last = [(t + i) % a.vocab for t in last for i in range(a.samples)]  # each continues with another token
    out = [[t] for t in last]
    for _ in range(a.tokens - 1):
        last = [int(np.argmax(x[-1])) for x in model.step(seqs, [[t] for t in last])]
        for o, t in zip(out, last):
            o.append(t)
    t2 = time.perf_counter()
    print(f"prompts: {a.sequences * a.prompt / (t1 - t0):.0f} tokens/s   decoding: {len(seqs) * max(1, a.tokens - 1) / (t2 - t1):.0f} tokens/s   first tokens: {[o[:6] for o in out]}")
    model.close()
    ctx.close()


if __name__ == "__main__":
    main()
