"""Attention over a paged key/value cache: what lies between the quantized projections of a decoder layer.

    QkNormRope       q, k, v of the projections: norms of q and k per head, rotation by position, rounding to bf16; k and v go into the cache
    PromptAttention  causal attention over whole prompts, packed one behind the other
    TreeAttention    attention of a decoded token, or of a chain or tree of drafted ones, over each sequence's cache
    KvCache          pages of keys and values: sequences that grow, fork, are cut back and freed; drafts that are kept move up.  Forks share pages until
                     one of them is to write there

The first three bind their buffers once (shapes and types are checked then) and are run once per step: ``op.run(stream)`` is one native
call that only enqueues.  Lengths, tables and masks are device arrays read when the kernel runs, so a recorded step
(``CudaContext.graph_begin``) serves a growing cache.  All tensors are ``DeviceTensor``; the arithmetic is described in include/wfb200.h.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence as Seq, Tuple

import numpy as np

from . import _native as N
from .backend import CudaContext, DeviceTensor, UnsupportedOperationError


def rope_table(rows: int, rot_dim: int, base: float = 10000.0, factors: Optional[np.ndarray] = None, scale: float = 1.0) -> np.ndarray:
    """fp32 [rows, rot_dim / 2, 2]: cosine and sine of position * base^(-2i / rot_dim) / factors[i], times `scale`, computed in
    64 bits (a GGUF model's rope_freqs are such factors)."""
    if rot_dim % 2 or rows < 0:
        raise ValueError(f"rope table of {rows} rows for rot_dim {rot_dim}")
    freq = base ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / max(rot_dim, 1))
    if factors is not None:
        freq = freq / np.asarray(factors, np.float64)
    angle = np.arange(rows, dtype=np.float64)[:, None] * freq[None, :]
    return (np.stack((np.cos(angle), np.sin(angle)), -1) * scale).astype(np.float32)


def _typed(name: str, t: Optional[DeviceTensor], dtype: str, *dims) -> int:
    """The address of `t`, which has this type and these dimensions (None: any); 0 where there is no tensor."""
    if t is None:
        return 0
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    shape = t.shape()
    if len(shape) != len(dims) or any(d is not None and d != s for d, s in zip(dims, shape)):
        raise ValueError(f"{name} must have the shape {tuple('*' if d is None else d for d in dims)}, got {shape}")
    return t.ptr


def _dense(name: str, t: DeviceTensor) -> None:
    if t.row_stride and t.row_stride != int(np.prod(t.shape()[1:])):
        raise UnsupportedOperationError(f"{name} must be without gaps")


def _stride(t: DeviceTensor) -> int:
    return t.row_stride or int(np.prod(t.shape()[1:]))


def _cache_args(keys: DeviceTensor, values: DeviceTensor, layers: int = 1) -> N.KvCacheArgs:
    """keys, values: [tokens, kv_heads, dim] (packed), [pages, kv_heads, page_tokens, dim] or the same with a first dimension of layers."""
    shape = keys.shape()
    if len(shape) not in (3, 4, 5):
        raise ValueError(f"keys must have 3 (packed), 4 (pages) or 5 (layers of pages) dimensions, got {shape}")
    for name, t in (("keys", keys), ("values", values)):
        _typed(name, t, "bf16", *shape)
        _dense(name, t)
    if len(shape) == 3:
        layers, pages, heads, page, dim = 1, shape[0], shape[1], 1, shape[2]
    else:
        layers, pages, heads, page, dim = (1, *shape) if len(shape) == 4 else shape
    return N.KvCacheArgs(keys.ptr, values.ptr, pages, layers, heads, page, dim)


class _Bound:
    """An operator with its buffers; they are kept alive with it."""

    def __init__(self, context: CudaContext, function: str, args, cache: N.KvCacheArgs, layer: int, tensors):
        self.context, self.args, self.cache, self.layer, self._tensors = context, args, cache, layer, tensors
        self._name, self._fn = function, getattr(context._lib, function)
        self._args, self._cache = ctypes.byref(args), ctypes.byref(cache)

    def run(self, stream: int = 0) -> None:
        rc = self._fn(self.context.handle, self._args, self._cache, self.layer, stream)
        if rc:
            self.context._ck(self._name, rc)


class QkNormRope(_Bound):
    """q [tokens, q_heads, dim], k and v [tokens, kv_heads, dim], fp32 or bf16, tokens any distance apart (q | k | v of one buffer);
    q_out bf16 [tokens, q_heads, dim].  keys, values: pages of the cache, or packed tensors.  positions i32 [tokens] are rows of `table`
    f32 [rows, rot_dim / 2, 2] (rope_table); slots i64 [tokens] = page * page_tokens + row, negative: not stored, None: slot i
    for token i.  pairs: "half" rotates (i, i + rot_dim / 2), "adjacent" (2i, 2i + 1).  q, or k and v, may be None."""

    def __init__(self, context: CudaContext, q, k, v, q_out, keys, values, positions, table, *, slots=None, norm: bool = False, gamma_q=None, gamma_k=None,
                 eps: float = 1e-5, pairs: str = "half", layer: int = 0):
        if pairs not in ("half", "adjacent"):
            raise ValueError(f"pairs must be 'half' or 'adjacent', got {pairs!r}")
        if (q is None) != (q_out is None) or (k is None) != (v is None) or (q is None and k is None):
            raise ValueError("q with q_out, k with v, or both")
        cache = _cache_args(keys, values)
        dim, first = cache.head_dim, q if q is not None else k
        tokens, dtype = first.shape()[0], first.dtype
        kind = {"f32": N.WF_DTYPE_F32, "bf16": N.WF_DTYPE_BF16}.get(dtype)
        if kind is None:
            raise UnsupportedOperationError(f"dtype {dtype} not supported")
        a = N.QkNormRopeArgs(tokens=tokens, x_dtype=kind, eps=eps, flags=(N.WF_QK_NORM if norm else 0) | (N.WF_ROPE_ADJACENT if pairs == "adjacent" else 0))
        a.q_dev = _typed("q", q, dtype, tokens, None, dim)
        a.k_dev, a.v_dev = (_typed(n, t, dtype, tokens, cache.kv_heads, dim) for n, t in (("k", k), ("v", v)))
        a.q_stride, a.k_stride, a.v_stride = (0 if t is None else _stride(t) for t in (q, k, v))
        if q is not None:
            a.q_heads = q.shape()[1]
            a.q_out_dev = _typed("q_out", q_out, "bf16", *q.shape())
            _dense("q_out", q_out)
        a.gamma_q_dev, a.gamma_k_dev = (_typed(n, t, "f32", dim) for n, t in (("gamma_q", gamma_q), ("gamma_k", gamma_k)))
        if not norm and (gamma_q is not None or gamma_k is not None):
            raise ValueError("gamma without norm")
        if table is not None:
            a.rope_dev = _typed("table", table, "f32", None, None, 2)
            a.rope_rows, a.rot_dim = table.shape()[0], 2 * table.shape()[1]
            a.positions_dev = _typed("positions", positions, "i32", tokens)
        a.slots_dev = _typed("slots", slots, "i64", tokens)
        super().__init__(context, "wf_qk_norm_rope", a, cache, layer, (q, k, v, q_out, keys, values, positions, table, slots, gamma_q, gamma_k))


class PromptAttention(_Bound):
    """q bf16 [tokens, q_heads, dim] (tokens may lie further apart), out bf16 [tokens, q_heads, dim], q_offsets i32 [seqs + 1].  keys and
    values packed [tokens, kv_heads, dim], or pages with tables i32 [seqs, width] and k_lens i32 [seqs] (past and prompt together)."""

    def __init__(self, context: CudaContext, q, keys, values, out, q_offsets, *, tables=None, k_lens=None, scale: Optional[float] = None, layer: int = 0):
        cache = _cache_args(keys, values)
        dim = cache.head_dim
        tokens, heads = q.shape()[:2]
        a = N.PromptAttentionArgs(tokens=tokens, q_heads=heads, seqs=q_offsets.shape()[0] - 1, scale=1 / math.sqrt(dim) if scale is None else scale)
        a.q_dev, a.out_dev, a.q_stride = _typed("q", q, "bf16", tokens, heads, dim), _typed("out", out, "bf16", tokens, heads, dim), _stride(q)
        _dense("out", out)
        a.q_offsets_dev = _typed("q_offsets", q_offsets, "i32", None)
        a.tables_dev, a.k_lens_dev = _typed("tables", tables, "i32", a.seqs, None), _typed("k_lens", k_lens, "i32", a.seqs)
        a.table_stride = 0 if tables is None else tables.shape()[1]
        super().__init__(context, "wf_prompt_attention", a, cache, layer, (q, keys, values, out, q_offsets, tables, k_lens))


class TreeAttention(_Bound):
    """q, out bf16 [tokens, q_heads, dim]: the new tokens of all sequences.  context i32 [seqs] tokens lie before them in the pages that
    tables i32 [seqs, width] name.  q_offsets i32 [seqs + 1], or None where every sequence has max_drafts; ancestors i64 [tokens], bit
    j: sees new token j (None: a chain).  max_context and max_drafts are upper bounds (of the whole decoding, if a recorded step serves it)."""

    def __init__(self, context: CudaContext, q, keys, values, out, tables, context_lens, *, max_context: int, q_offsets=None, max_drafts: int = 1, ancestors=None,
                 scale: Optional[float] = None, layer: int = 0):
        cache = _cache_args(keys, values)
        dim = cache.head_dim
        tokens, heads = q.shape()[:2]
        seqs = context_lens.shape()[0]
        a = N.TreeAttentionArgs(tokens=tokens, q_heads=heads, seqs=seqs, max_drafts=max_drafts, max_context=max_context,
                                scale=1 / math.sqrt(dim) if scale is None else scale)
        a.q_dev, a.out_dev, a.q_stride = _typed("q", q, "bf16", tokens, heads, dim), _typed("out", out, "bf16", tokens, heads, dim), _stride(q)
        _dense("out", out)
        a.q_offsets_dev = _typed("q_offsets", q_offsets, "i32", seqs + 1)
        a.tables_dev, a.table_stride = _typed("tables", tables, "i32", seqs, None), tables.shape()[1]
        a.context_dev, a.ancestors_dev = _typed("context_lens", context_lens, "i32", seqs), _typed("ancestors", ancestors, "i64", tokens)
        super().__init__(context, "wf_tree_attention", a, cache, layer, (q, keys, values, out, tables, context_lens, q_offsets, ancestors))


class Sequence:
    """Tokens of one sequence in a KvCache: how many, and the pages that hold them."""

    def __init__(self, cache: "KvCache", pages: List[int], tokens: int):
        self.cache, self.pages, self.tokens = cache, pages, tokens

    def extend(self, n: int, stream: int = 0) -> List[int]:
        """Room for n more tokens; their slots (page * page_tokens + row), in pages that are this sequence's alone: a part-full last page that others hold
        too is replaced by a copy of the rows in use (on `stream`, the one that the slots will be written on)."""
        if n < 0:
            raise ValueError(f"extend by {n} tokens")
        c, size = self.cache, self.cache.page_tokens
        end = self.tokens + n
        self.pages += c._own([self], [(self.tokens, end)], max(0, -(-end // size) - len(self.pages)), stream)
        slots = [self.pages[t // size] * size + t % size for t in range(self.tokens, end)]
        self.tokens = end
        return slots

    def truncate(self, tokens: int) -> None:
        """Forget what lies behind the first `tokens` (drafts that were not kept); pages that hold nothing any more are given back."""
        if not 0 <= tokens <= self.tokens:
            raise ValueError(f"{tokens} of {self.tokens} tokens")
        keep = -(-tokens // self.cache.page_tokens)
        self.cache._release(self.pages[keep:])
        self.pages, self.tokens = self.pages[:keep], tokens

    def fork(self, stream: int = 0) -> "Sequence":
        """A sequence with the same tokens: whole pages are shared, the last one, if it is part full, is copied (on `stream`)."""
        return self.cache.fork([self], stream)[0]

    def free(self) -> None:
        self.truncate(0)


class KvCache:
    """`pages` pages of page_tokens tokens for every layer: keys and values bf16 [layers, pages, kv_heads, page_tokens, head_dim], allocated here or
    given.  Page numbers are handed out by the native pool (wf_pages_*), which counts the sequences that hold each."""

    def __init__(self, context: CudaContext, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int, keys: Optional[DeviceTensor] = None,
                 values: Optional[DeviceTensor] = None):
        if (keys is None) != (values is None):
            raise ValueError("keys and values, or neither")
        if min(layers, pages, page_tokens, kv_heads, head_dim) < 1:
            raise ValueError(f"a cache of {layers} layers, {pages} pages of {page_tokens} tokens, {kv_heads} heads of {head_dim}")
        shape = (layers, pages, kv_heads, page_tokens, head_dim)
        self.context, self.layers, self.page_count, self.page_tokens, self.kv_heads, self.head_dim = context, layers, pages, page_tokens, kv_heads, head_dim
        self._owned, self._pool = [], 0
        self._fork_arrays = {}  # stream: device arrays of its forks (pairs, rows, how many fit)
        try:
            if keys is None:
                for _ in range(2):
                    self._owned.append(context.allocate(int(np.prod(shape)) * 2))
                keys, values = (DeviceTensor(p, shape, "bf16", owner=context) for p in self._owned)
            self.keys, self.values = keys, values
            for name, t in (("keys", keys), ("values", values)):
                _typed(name, t, "bf16", *shape)
            self._args = _cache_args(keys, values)
            self._ref = ctypes.byref(self._args)
            pool = ctypes.c_int64()
            N.check("wf_pages_create", context._lib.wf_pages_create(pages, ctypes.byref(pool)))
        except BaseException:
            for p in self._owned:
                context.free(p)
            raise
        self._pool = pool.value

    # ---- pages
    def _ids(self, ids: Seq[int]):
        return (ctypes.c_int32 * len(ids))(*ids)

    def _take(self, n: int) -> List[int]:
        out = (ctypes.c_int32 * n)()
        N.check("wf_pages_take", self.context._lib.wf_pages_take(self._pool, n, out))
        return list(out)

    def _share(self, ids: Seq[int]) -> None:
        N.check("wf_pages_share", self.context._lib.wf_pages_share(self._pool, len(ids), self._ids(ids)))

    def _release(self, ids: Seq[int]) -> None:
        N.check("wf_pages_release", self.context._lib.wf_pages_release(self._pool, len(ids), self._ids(ids)))

    def free_pages(self) -> int:
        n = ctypes.c_int64()
        N.check("wf_pages_info", self.context._lib.wf_pages_info(self._pool, None, ctypes.byref(n)))
        return n.value

    def holders(self, page: int) -> int:
        n = ctypes.c_int64()
        N.check("wf_pages_holders", self.context._lib.wf_pages_holders(self._pool, page, ctypes.byref(n)))
        return n.value

    # ---- sequences
    def sequence(self) -> Sequence:
        return Sequence(self, [], 0)

    def tables(self, sequences: Seq[Sequence], width: Optional[int] = None) -> np.ndarray:
        """i32 [len(sequences), width]: the page tables that the operators read."""
        width = max([1] + [len(s.pages) for s in sequences]) if width is None else width
        out = np.zeros((len(sequences), width), np.int32)
        for row, s in zip(out, sequences):
            if len(s.pages) > width:
                raise ValueError(f"a sequence of {len(s.pages)} pages in tables of {width}")
            row[:len(s.pages)] = s.pages
        return out

    def fork(self, sequences: Seq[Sequence], stream: int = 0) -> List[Sequence]:
        """A second sequence for each, with the same tokens: whole pages shared, part-full last pages copied, all in one call on `stream`."""
        part = [s for s in sequences if s.tokens % self.page_tokens]
        shared = [p for s in sequences for p in s.pages[:s.tokens // self.page_tokens]]
        self._share(shared)
        try:
            fresh = self._take(len(part))
        except BaseException:
            self._release(shared)
            raise
        out, pairs, rows = [], [], []
        for s in sequences:
            whole, rest = divmod(s.tokens, self.page_tokens)
            pages = s.pages[:whole]
            if rest:
                pages = pages + [fresh[len(pairs)]]
                pairs.append((s.pages[whole], pages[-1]))
                rows.append(rest)
            out.append(Sequence(self, pages, s.tokens))
        try:
            self._copy_rows(pairs, rows, stream)
        except BaseException:
            self._release(shared + fresh)
            raise
        return out

    def own(self, sequences: Seq[Sequence], spans: Seq[Tuple[int, int]], stream: int = 0) -> None:
        """Before tokens [start, stop) of each sequence are written to (``compact``): pages of them that other sequences hold too are replaced by copies of the
        rows in use, all in one call on `stream`.  Tables made before this name the old pages."""
        self._own(sequences, spans, 0, stream)

    def _own(self, sequences: Seq[Sequence], spans, more: int, stream: int) -> List[int]:
        """Pages that hold tokens [spans[i][0], spans[i][1]) of a sequence and have other holders too are replaced by copies; `more` free pages besides, which
        are returned.  All or nothing."""
        size, places, left = self.page_tokens, [], {}
        for s, (start, stop) in zip(sequences, spans):
            for i in range(start // size, min(len(s.pages), -(-stop // size))) if start < stop else ():
                page = s.pages[i]
                left.setdefault(page, self.holders(page))
                if left[page] > 1:
                    left[page] -= 1
                    places.append((s, i))
        fresh = self._take(len(places) + more)
        try:
            self._copy_rows([(s.pages[i], page) for (s, i), page in zip(places, fresh)], [min(size, s.tokens - i * size) for s, i in places], stream)
        except BaseException:
            self._release(fresh)
            raise
        self._release([s.pages[i] for s, i in places])
        for (s, i), page in zip(places, fresh):
            s.pages[i] = page
        return fresh[len(places):]

    def _copy_rows(self, pairs, rows, stream: int) -> None:
        """copy_pages of page numbers that the host has."""
        if pairs:
            to, counts = self._arrays(len(pairs), stream)
            self.context.copy_to_device(to, np.array(pairs, np.int32), stream)
            self.context.copy_to_device(counts, np.array(rows, np.int32), stream)
            self.copy_pages(DeviceTensor(to, (len(pairs), 2), "i32"), DeviceTensor(counts, (len(rows),), "i32"), stream)

    def _arrays(self, n: int, stream: int):
        """Device arrays for the pairs and rows of n copies on this stream; the old ones stay until larger ones are there."""
        ctx, (to, counts, room) = self.context, self._fork_arrays.get(stream, (0, 0, 0))
        if n > room:
            old, room = [p for p in (to, counts) if p], max(16, 2 * n)
            to = ctx.allocate(room * 8)
            try:
                counts = ctx.allocate(room * 4)
            except BaseException:
                ctx.free(to)
                raise
            self._fork_arrays[stream] = to, counts, room
            for p in old:
                ctx.free(p)
        return to, counts

    def layer(self, i: int):
        """keys and values of one layer, bf16 [pages, kv_heads, page_tokens, head_dim]."""
        if not 0 <= i < self.layers:
            raise ValueError(f"layer {i} of {self.layers}")
        shape = self.keys.shape()[1:]
        skip = i * int(np.prod(shape)) * 2
        return tuple(DeviceTensor(t.ptr + skip, shape, "bf16", owner=t) for t in (self.keys, self.values))

    # ---- device
    def copy_pages(self, pairs: DeviceTensor, rows: Optional[DeviceTensor] = None, stream: int = 0) -> None:
        """In every layer page pairs[i][0] to page pairs[i][1] (i32 [n, 2]), the first rows[i] tokens of it (i32 [n]; None: all)."""
        n = pairs.shape()[0]
        ctx = self.context
        ctx._ck("wf_cache_copy_pages", ctx._lib.wf_cache_copy_pages(ctx.handle, self._ref, _typed("pairs", pairs, "i32", n, 2), _typed("rows", rows, "i32", n), n, stream))

    def compact(self, tables: DeviceTensor, context_lens: DeviceTensor, kept: DeviceTensor, counts: DeviceTensor, stream: int = 0) -> None:
        """In every layer token context_lens[s] + kept[s][i] of sequence s becomes token context_lens[s] + i, i < counts[s]; kept i32
        [seqs, most] ascending.  The pages that tokens move to have to be the sequence's alone (``own``)."""
        seqs, most = kept.shape()
        ctx = self.context
        ctx._ck("wf_cache_compact", ctx._lib.wf_cache_compact(
            ctx.handle, self._ref, _typed("tables", tables, "i32", seqs, None), tables.shape()[1], _typed("context_lens", context_lens, "i32", seqs),
            _typed("kept", kept, "i32", seqs, most), most, _typed("counts", counts, "i32", seqs), seqs, stream))

    def close(self) -> None:
        if self._pool:
            pool, self._pool = self._pool, 0
            N.check("wf_pages_destroy", self.context._lib.wf_pages_destroy(pool))
            for p in self._owned + [p for arrays in self._fork_arrays.values() for p in arrays[:2]]:
                if self.context.handle:
                    self.context.free(p)
            self._owned, self._fork_arrays = [], {}
