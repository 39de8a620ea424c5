"""Workloads of attention that does not read every key of every sequence: what a program that serves long contexts does with the paged key/value cache.

`listed()` names twelve, `draw(rng)` makes more of the same ranges.  A case is one of these kinds:

  bounds    the largest and smallest element of the keys of a page, for every dimension, in 8 bits: of the pages that new tokens went to, in all layers
  select    which pages a new token reads: for every token and kv head those whose bounds promise the largest scores, the first ones and the last ones
  selected  attention of new tokens over such lists of pages
  shared    attention of new tokens where sequences have a long prefix in common, whose keys are read once for all of them

Lengths are texts, one number for each sequence (or group of sequences).  A cache holds bf16 [layers, pages, kv_heads, page_tokens, dim]; token t of a
sequence lies in row t % page_tokens of page tables[sequence, t // page_tokens].  New tokens lie behind a sequence's context: one, a chain, or a tree of drafted
ones in which each sees the context and its own ancestors.
"""
from __future__ import annotations

import itertools
import math

import torch

own = False  # True: the framework's operators; False: the same from elementary operations

MAX_KEYS = 600 << 20    # bytes of keys and values that a drawn attention case reads
MAX_GATHER = 6 << 30    # bytes that the plain form of a drawn case may gather
DRAFTS = 64             # drafted tokens of a sequence, at most: a mask is one 64-bit word
LEAST_EXPONENT = -60    # of a scale: products of two are normal numbers


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    batch = ",".join(str(500 + 331 * i + (i * i * 37) % 900) for i in range(48))  # contexts from 500 to 16,000
    return [
        # Sixteen sequences have each decoded a token: the page that it went to, in 32 layers.  The smallest call.
        dict(name="bounds_step", kind="bounds", layers=32, lens=",".join(str(100 + 77 * i) for i in range(16)), new="1" + ",1" * 15, kv_heads=8, dim=128, page=64),
        # An 8192-token prompt has gone through 32 layers.
        dict(name="bounds_prompt", kind="bounds", layers=32, lens="8192", new="8192", kv_heads=8, dim=128, page=64),
        # Prompts of odd lengths behind pasts, heads of 96, small pages.
        dict(name="bounds_ragged", kind="bounds", layers=9, lens="1511,40,903,2999,1,640,0,1777", new="1000,37,1,513,1,0,0,770", kv_heads=5, dim=96, page=16),
        # One decoded token at a context of 32,000: 64 of 500 pages.
        dict(name="select_1tok", kind="select", lens="32000", drafts="1", shape="single", q_heads=32, kv_heads=8, dim=128, page=64, width=64, first=1, recent=128),
        # A batch of sequences of the 70B-shape model's heads.
        dict(name="select_batch", kind="select", lens=batch, drafts="1" + ",1" * 47, shape="single", q_heads=64, kv_heads=8, dim=128, page=64, width=64, first=1, recent=128),
        # A tree of drafted tokens at a very long context in small pages.
        dict(name="select_tree_long", kind="select", lens="131059", drafts="21", shape="tree", q_heads=24, kv_heads=8, dim=96, page=16, width=256, first=4, recent=256),
        # One decoded token reads 64 pages of 64 tokens.
        dict(name="selected_1tok", kind="selected", lens="32000", drafts="1", shape="single", q_heads=32, kv_heads=8, dim=128, page=64, width=64, first=1, recent=128),
        # The batch of above; the shortest contexts have fewer pages than the lists have room for.
        dict(name="selected_batch", kind="selected", lens=batch, drafts="1" + ",1" * 47, shape="single", q_heads=64, kv_heads=8, dim=128, page=64, width=32, first=1, recent=128),
        # Trees of drafted tokens of several sequences, heads of 80, an odd group, small pages, one sequence without a context.
        dict(name="selected_trees", kind="selected", lens="3511,2040,0,7999,1", drafts="9,16,5,17,1", shape="tree", q_heads=20, kv_heads=4, dim=80, page=16, width=96, first=1, recent=64),
        # Four samples of one prompt.
        dict(name="shared_4", kind="shared", members="4", prefix="1024", lens="40,77,12,129", drafts="1,1,1,1", shape="single", q_heads=32, kv_heads=8, dim=128, page=64),
        # Sixty-four requests behind one long instruction, 70B-shape heads.  The largest call.
        dict(name="shared_64", kind="shared", members="64", prefix="16384", lens=",".join(str(20 + (53 * i * i) % 391) for i in range(64)), drafts="1" + ",1" * 63,
             shape="single", q_heads=64, kv_heads=8, dim=128, page=64),
        # Groups of several sizes, one sequence that shares nothing, trees of drafted tokens, heads of 64.
        dict(name="shared_groups", kind="shared", members="9,1,5,2", prefix="3008,0,512,8000", lens="100,7,0,311,64,65,1,900,30,1777,5,50,500,2,33,640,641", drafts="5,1,7,5,5,12,1,5,3,5,5,6,1,9,5,4,8",
             shape="tree", q_heads=24, kv_heads=8, dim=64, page=32),
    ]


def _log(rng, lo, hi):
    return lo * (hi / lo) ** rng.random()


def _heads(rng):
    kv = rng.choice((1, 2, 4, 8, 8, 16))
    group = rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 16) if kv * g <= 64])
    return kv * group, kv


def _texts(values):
    return ",".join(map(str, values))


def draw(rng):
    kind = rng.choice(("bounds", "select", "select", "selected", "selected", "shared", "shared"))
    q_heads, kv_heads = _heads(rng)
    dim = rng.choice((64, 64, 128, 128, 128, 80, 96, 112))
    page = rng.choice((16, 32, 64, 128))
    if kind == "bounds":
        layers = rng.randint(1, 48)
        seqs = max(1, int(_log(rng, 1, 48)))
        prompts = rng.random() < 0.5
        lens = [int(_log(rng, 1, 8192 if prompts else 2000)) for _ in range(seqs)]
        while layers * sum(-(-n // page) * page + page for n in lens) * kv_heads * dim * 4 > 1 << 30:
            lens, layers = [max(1, n // 2) for n in lens], (layers + 1) // 2
        new = [rng.randint(i == 0, n) if prompts else 1 for i, n in enumerate(lens)]
        return dict(kind="bounds", layers=layers, lens=_texts(lens), new=_texts(new), kv_heads=kv_heads, dim=dim, page=page)
    shape = rng.choice(("single", "single", "chain", "tree"))
    most_drafts = {"single": 1, "chain": 8, "tree": 24}[shape]
    if kind != "shared":
        seqs = max(1, int(_log(rng, 1, 48)))
        drafts = [1 if shape == "single" else rng.randint(1, most_drafts) for _ in range(seqs)]
        top = _log(rng, 64, 131072)
        lens = [int(_log(rng, max(1, top / 8), top)) for _ in range(seqs)]
        first, recent = rng.randint(0, 4), rng.choice((0, 1, 64, 100, 256))
        tail = (recent + max(drafts) + page - 2) // page + 2
        width = first + tail + int(_log(rng, 1, 8192 / page))
        if kind == "select":
            # the plain form's codes as fp32 numbers, and its scores, padded to the longest
            while seqs * (max(lens) // page + 1) * kv_heads * (2 * dim + max(drafts) * q_heads // kv_heads) * 12 > MAX_GATHER:
                lens = [max(1, n // 2) for n in lens]
        else:
            while sum(drafts) * kv_heads * width * page * dim * 4 > MAX_KEYS and width > first + tail + 1:
                width = first + tail + (width - first - tail) // 2
            while seqs > 1 and (sum(drafts) * kv_heads * width * page * dim * 4 > 2 * MAX_KEYS or sum(lens) * kv_heads * dim * 4 > 3 << 30):
                seqs = seqs // 2
                lens, drafts = lens[:seqs], drafts[:seqs]
        return dict(kind=kind, lens=_texts(lens), drafts=_texts(drafts), shape=shape, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, width=width, first=first, recent=recent)
    members = [max(1, int(_log(rng, 1, 64))) for _ in range(rng.choice((1, 1, 2, rng.randint(3, 6))))]
    while sum(members) > 64:
        members[members.index(max(members))] //= 2
    top = _log(rng, page, 16384)
    prefix = [0 if n == 1 else int(_log(rng, max(1, top / 8), top)) // page * page for n in members]
    own_top = _log(rng, 1, 1000)
    lens = [int(_log(rng, 1, own_top)) - (rng.random() < 0.1) for _ in range(sum(members))]
    drafts = [1 if shape == "single" else rng.randint(1, most_drafts) for _ in lens]
    # what the plain form gathers, padded to the longest, and its scores
    while len(lens) * (max(prefix) + max(lens) + max(drafts)) * (kv_heads * dim * 16 + q_heads * max(drafts) * 8) > MAX_GATHER:
        prefix, lens = [n // 2 // page * page for n in prefix], [n // 2 for n in lens]
    return dict(kind="shared", members=_texts(members), prefix=_texts(prefix), lens=_texts(lens), drafts=_texts(drafts), shape=shape, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page)


# ------------------------------------------------------------------------------------------------ inputs
def _ints(text):
    return [int(n) for n in text.split(",")] if text else []


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _offsets(lens):
    return list(itertools.accumulate(lens, initial=0))


def _pages(totals, page, gen, spare=3):
    """Page tables for sequences of `totals` tokens, over pages in random order; as many pages and `spare` more."""
    need = [-(-n // page) for n in totals]
    order = torch.randperm(sum(need) + spare, device="cuda", generator=gen).to(torch.int32)
    width = max(1, max(need))
    at = torch.tensor(_offsets(need)[:-1], device="cuda")[:, None] + torch.arange(width, device="cuda")[None, :]
    inside = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    return torch.where(inside, order[at.clamp(max=order.numel() - 1)], 0).contiguous(), order.numel()


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.bfloat16) * scale


def _ancestors(n, shape, generator):
    """Which drafted tokens each of n sees, itself among them, as the bits of a word."""
    words, mask = [], (1 << 64) - 1
    for i in range(n):
        parent = -1 if i == 0 else i - 1 if shape != "tree" else int(torch.randint(max(0, i - 6), i, (1,), generator=generator))
        words.append((1 << i) | (words[parent] if parent >= 0 else 0))
    return [w - (1 << 64) if w >> 63 else w & mask for w in words]


def _spans(c, n, m):
    """Of a sequence with a context of n tokens and m new ones: its pages, the first of those that every list has at its end, how many of those before that one a list has room for."""
    last = -(-(n + m) // c["page"])
    tail = max(0, n - c["recent"]) // c["page"]
    return last, tail, min(max(0, tail - c["first"]), c["width"] - min(c["first"], tail) - (last - tail))


def prepare(case, seed):
    gen, c = _gen(seed), case
    host = torch.Generator().manual_seed(seed)
    s = {"case": c}
    hk, d, page = c["kv_heads"], c["dim"], c["page"]
    lens = _ints(c["lens"])
    if c["kind"] == "bounds":
        s["tables"], pages = _pages(lens, page, gen)
        s.update(first=_i32([n - m for n, m in zip(lens, _ints(c["new"]))]), stop=_i32(lens))
        # keys have directions that all of a sequence share, and some large dimensions
        s["keys"] = _normal(gen, c["layers"], pages, hk, page, d) * (0.3 + 2 * torch.rand(d, device="cuda", generator=gen).bfloat16() ** 4)
        s["values"] = torch.empty_like(s["keys"])
        s["codes"] = torch.randint(-127, 128, (c["layers"], pages, hk, 2, d), device="cuda", generator=gen, dtype=torch.int8)
        s["scales"] = torch.full((c["layers"], pages, hk), 2.0**-6, device="cuda")
        s["stream"] = torch.cuda.Stream()
        return s
    drafts, hq = _ints(c["drafts"]), c["q_heads"]
    s.update(q=_normal(gen, sum(drafts), hq, d, scale=1.5), q_offsets=_i32(_offsets(drafts)), scale=1 / math.sqrt(d))
    s["ancestors"] = torch.tensor([w for n in drafts for w in _ancestors(n, c["shape"], host)], dtype=torch.int64, device="cuda")
    if c["kind"] == "shared":
        members, prefix = _ints(c["members"]), _ints(c["prefix"])
        of = [g for g, n in enumerate(members) for _ in range(n)]
        own_tables, pages = _pages([n + m for n, m in zip(lens, drafts)], page, gen)
        shared_tables, more = _pages(prefix, page, gen)
        width = max(prefix[g] // page for g in of) + own_tables.shape[1]
        at = torch.arange(width, device="cuda")[None, :]
        begin = (_i32(prefix) // page)[_i32(of).long()][:, None].long()
        s["tables"] = torch.where(at < begin, shared_tables[_i32(of).long()].gather(1, at.expand(len(of), -1).clamp(max=shared_tables.shape[1] - 1)) + pages,
                                  own_tables.gather(1, (at - begin).clamp(0, own_tables.shape[1] - 1))).contiguous()
        pages += more
        s.update(groups=_i32(_offsets(members)), prefix=_i32(prefix), context=_i32([prefix[g] + n for g, n in zip(of, lens)]))
    else:
        s["tables"], pages = _pages([n + m for n, m in zip(lens, drafts)], page, gen)
        s["context"] = _i32(lens)
        lists = (sum(drafts), hk, c["width"])
        if c["kind"] == "select":
            # bounds of keys: an interval around a middle that some pages share with the queries
            middle = torch.randint(-60, 61, (pages, hk, 1, d), device="cuda", generator=gen, dtype=torch.int16)
            half = torch.randint(10, 67, (pages, hk, 1, d), device="cuda", generator=gen, dtype=torch.int16)
            s["codes"] = torch.cat((middle + half, middle - half), 2).to(torch.int8)
            s["scales"] = 2.0 ** torch.randint(-7, -4, (pages, hk), device="cuda", generator=gen).float()
            s.update(pages=torch.empty(lists, device="cuda", dtype=torch.int32), lens=torch.empty(*lists[:2], 2, device="cuda", dtype=torch.int32))
            return s
        # lists as a selection makes them; the tokens of a sequence agree about three quarters of the pages
        s["pages"] = torch.full(lists, -1, device="cuda", dtype=torch.int32)
        lens_of = torch.zeros(*lists[:2], 2, dtype=torch.int32)
        for i, (n, m, row) in enumerate(zip(lens, drafts, _offsets(drafts))):
            last, tail, k = _spans(c, n, m)
            first, between = min(c["first"], tail), max(0, tail - c["first"])
            liked = torch.rand(1, hk, between, device="cuda", generator=gen).expand(m, -1, -1)
            liked = torch.where(torch.rand(m, hk, between, device="cuda", generator=gen) < 0.25, torch.rand(m, hk, between, device="cuda", generator=gen), liked)
            which = first + liked.topk(k, -1).indices.sort(-1).values
            ends = [torch.arange(*r, device="cuda").expand(m, hk, -1) for r in ((0, first), (tail, last))]
            which = torch.cat((ends[0], which, ends[1]), -1)
            s["pages"][row:row + m, :, :which.shape[-1]] = s["tables"][i][which]
            lens_of[row:row + m, :, 0] = n - page * (between - k)
            lens_of[row:row + m, :, 1] = lens_of[row:row + m, :, 0] + (m if c["shape"] == "tree" else torch.arange(1, m + 1, dtype=torch.int32)[:, None])
        s["lens"] = lens_of.cuda()
    s.update(keys=_normal(gen, pages, hk, page, d), values=_normal(gen, pages, hk, page, d), out=torch.empty_like(s["q"]))
    return s


# ------------------------------------------------------------------------------------------------ the framework's operators
_backend = None


def _context():
    """A program has one backend (one context, one stream) for its lifetime."""
    global _backend
    if _backend is None:
        from warpforge_b200.backend import NvidiaBackend

        _backend = NvidiaBackend(0)
    return _backend.cuda_context


def _held(t):
    """A torch tensor's memory as the framework's tensor."""
    from warpforge_b200.backend import DeviceTensor

    names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.int32: "i32", torch.int64: "i64", torch.int8: "i8"}
    return DeviceTensor(t.data_ptr(), tuple(t.shape), names[t.dtype], owner=t)


def _call(s):
    """The operator with its buffers bound, as a program keeps it for its loop."""
    from warpforge_b200 import attention

    c, ctx = s["case"], _context()
    h = {k: _held(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["kind"] == "bounds":
        cache = attention.KvCache(ctx, c["layers"], h["keys"].shape()[1], c["page"], c["kv_heads"], c["dim"], keys=h["keys"], values=h["values"])
        bounds = attention.PageBounds(cache, codes=h["codes"], scales=h["scales"])
        most = max(_ints(c["new"]))
        return lambda: bounds.update(h["tables"], h["first"], h["stop"], max_tokens=most, stream=s["stream"].cuda_stream)
    drafts = dict(q_offsets=h["q_offsets"], max_drafts=max(_ints(c["drafts"])))
    if c["kind"] == "select":
        return attention.SelectPages(ctx, h["q"], h["codes"], h["scales"], h["tables"], h["context"], h["pages"], h["lens"], page_tokens=c["page"], max_context=max(_ints(c["lens"])),
                                     first=c["first"], recent=c["recent"], tree=c["shape"] == "tree", **drafts).run
    words = h["ancestors"] if c["shape"] == "tree" else None
    if c["kind"] == "selected":
        return attention.SelectedAttention(ctx, h["q"], h["keys"], h["values"], h["out"], h["pages"], h["lens"], ancestors=words, scale=s["scale"]).run
    return attention.SharedPrefixAttention(ctx, h["q"], h["keys"], h["values"], h["out"], h["tables"], h["context"], h["groups"], h["prefix"], max_prefix=max(_ints(c["prefix"])),
                                           max_own=max(_ints(c["lens"])), ancestors=words, scale=s["scale"], **drafts).run


# ------------------------------------------------------------------------------------------------ their plain forms
def _power(e):
    """2^e as fp32, exactly, for the exponents of normal numbers."""
    return ((e + 127) << 23).view(torch.float32)


def _scale_for(size):
    """The least power of two of which 127 times is `size` or more, as fp32; +Inf where size is not finite.  size = f 2^k, f in [1/2, 1), and 127 = 0.9921875 2^7."""
    f, k = torch.frexp(size)
    e = torch.where(f > 0.9921875, k - 6, k - 7).clamp(min=LEAST_EXPONENT).to(torch.int32)
    return torch.where(size.isfinite(), _power(torch.where(size.isfinite() & (size > 0), e, LEAST_EXPONENT)), float("inf"))


def _plain_bounds(s):
    page = s["case"]["page"]
    index = torch.arange(s["tables"].shape[1], device="cuda")[None, :] * page
    first, stop = s["first"][:, None], s["stop"][:, None]
    touched = (first < stop) & (index < stop) & (index + page > first)
    which, rows = s["tables"][touched].long(), (stop - index).clamp(max=page)[touched]
    k = s["keys"][:, which].float()
    there = (torch.arange(page, device="cuda")[None, :] < rows[:, None])[None, :, None, :, None]
    hi, lo = torch.where(there, k, float("-inf")).amax(3), torch.where(there, k, float("inf")).amin(3)
    scale = _scale_for(torch.maximum(hi.abs(), lo.abs()).amax(-1))
    fine, by = scale.isfinite()[..., None], scale[..., None]
    s["codes"][:, which] = torch.stack((torch.where(fine, (hi / by).ceil(), 0.0), torch.where(fine, (lo / by).floor(), 0.0)), 3).to(torch.int8)
    s["scales"][:, which] = scale


def _rows(s):
    """Sequence and place in it of every new token, and which rows a sequence's new tokens are, padded to the most."""
    start = s["q_offsets"][:-1].long()
    count = s["q_offsets"][1:].long() - start
    tokens = s["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(start), device="cuda"), count, output_size=tokens)
    widest = max(_ints(s["case"]["drafts"]))
    row = (start[:, None] + torch.arange(widest, device="cuda")[None, :]).clamp(max=tokens - 1)
    return seq, torch.arange(tokens, device="cuda") - start[seq], count, row


def _plain_select(s):
    c, q = s["case"], s["q"].float()
    hk, page, width = c["kv_heads"], c["page"], c["width"]
    seq, place, count, row = _rows(s)
    size = q.abs().amax(-1)
    by = _scale_for(size)
    q8 = torch.where(by.isfinite()[..., None], (q / by[..., None]).round(), 0.0)
    by = torch.where(by.isfinite(), by, 1.0)
    # [sequences, kv_heads, tokens * group, 2 dim] against the codes of the sequences' pages
    both = torch.cat((q8.clamp(min=0), q8.clamp(max=0)), -1)[row].unflatten(2, (hk, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    where = s["tables"].long()
    sums = both @ s["codes"][where].float().flatten(3).permute(0, 2, 3, 1)
    heads = sums.unflatten(2, (row.shape[1], -1)) * by[row].unflatten(2, (hk, -1)).permute(0, 2, 1, 3)[..., None]
    page_scale = s["scales"][where].permute(0, 2, 1)[:, :, None]
    scores = torch.where(page_scale.isfinite(), heads.amax(3) * torch.where(page_scale.isfinite(), page_scale, 1.0), float("inf"))
    scores = scores.transpose(1, 2)[seq, place]                                       # [tokens, kv_heads, pages]
    index = torch.arange(scores.shape[-1], device="cuda")
    context = s["context"].long()[seq]
    last = (context + count[seq] + page - 1) // page
    tail = (context - c["recent"]).clamp(min=0) // page
    first = tail.clamp(max=c["first"])
    between = tail - first
    k = torch.minimum(between, width - first - (last - tail))
    last, tail, first, k = (x[:, None, None] for x in (last, tail, first, k))
    inside = (index >= first) & (index < tail)
    order = torch.where(inside, scores, float("-inf")).sort(dim=-1, descending=True, stable=True).indices  # ties: the lowest first
    best = torch.zeros_like(order).scatter(2, order, index.expand_as(order)) < k
    chosen = (best & inside) | (index < first) | ((index >= tail) & (index < last))
    listed_ = (~chosen).to(torch.int8).sort(dim=-1, stable=True).indices                  # those that are chosen, ascending
    names = s["tables"][seq][:, None].expand(-1, hk, -1).gather(2, listed_)
    names = torch.where(index < chosen.sum(-1, keepdim=True), names, -1)[..., :width]
    s["pages"].fill_(-1)
    s["pages"][..., :names.shape[-1]] = names
    held = context - page * (between - k[:, 0, 0])
    keys = held + (count[seq] if c["shape"] == "tree" else place + 1)
    s["lens"].copy_(torch.stack((held, keys), -1)[:, None].expand(-1, hk, -1))


def _weights(scores, seen):
    """Softmax over the keys that a row sees, in place; rows that see none get zeros."""
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(torch.where(total == 0, 1.0, total))


def _plain_selected(s):
    c = s["case"]
    hk, page = c["kv_heads"], c["page"]
    held, keys = (s["lens"][..., i, None].long() for i in (0, 1))                      # [tokens, kv_heads, 1]
    at = torch.arange(c["width"] * page, device="cuda")
    head = torch.arange(hk, device="cuda")[None, :, None]
    where = s["pages"].long().clamp(min=0).repeat_interleave(page, -1)
    k, v = (x[where, head, at % page].float() for x in (s["keys"], s["values"]))       # [tokens, kv_heads, keys, dim]
    draft = at - held
    seen = (draft < 0) | (at < keys)
    if c["shape"] == "tree":
        seen = (draft < 0) | ((at < keys) & ((s["ancestors"][:, None, None] >> draft.clamp(0, 63)) & 1 == 1))
    queries = s["q"].float().unflatten(1, (hk, -1))
    w = _weights(queries @ k.transpose(2, 3) * s["scale"], seen[:, :, None].expand(-1, -1, queries.shape[2], -1))
    return (w @ v).flatten(1, 2).bfloat16()


def _plain_shared(s):
    c, q = s["case"], s["q"].float()
    hk, page = c["kv_heads"], c["page"]
    seq, place, count, row = _rows(s)
    of = torch.repeat_interleave(torch.arange(len(_ints(c["members"])), device="cuda"), s["groups"].diff().long(), output_size=len(_ints(c["lens"])))
    most = max(_ints(c["prefix"])[g] + n + m for g, n, m in zip([g for g, n in enumerate(_ints(c["members"])) for _ in range(n)], _ints(c["lens"]), _ints(c["drafts"])))
    at = torch.arange(most, device="cuda")
    first = s["tables"][s["groups"][:-1].long()[of]]                                   # the prefix lies in the pages of a group's first
    index = (at // page).clamp(max=s["tables"].shape[1] - 1)
    where = torch.where(at < s["prefix"][of][:, None], first[:, index], s["tables"][:, index]).long()
    k, v = (x[where, :, at % page].float().transpose(1, 2) for x in (s["keys"], s["values"]))
    queries = q[row].unflatten(2, (hk, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)       # [seqs, kv_heads, group * drafts, dim]
    draft = at[None, :] - s["context"].long()[:, None]
    bit = (s["ancestors"][row][:, :, None] >> draft.clamp(0, 63)[:, None, :]) & 1
    seen = (draft[:, None, :] < 0) | ((draft[:, None, :] < count[:, None, None]) & (draft[:, None, :] < DRAFTS) & (bit == 1))
    w = _weights(queries @ k.transpose(2, 3) * s["scale"], seen[:, None].repeat(1, 1, q.shape[1] // hk, 1))
    out = (w @ v).unflatten(2, (-1, row.shape[1])).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[seq, place].bfloat16()


def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        if "call" not in s:
            s["call"] = _call(s)
        s["call"]()
    if kind == "bounds":
        if own:
            with torch.cuda.stream(s["stream"]):
                return s["codes"] * s["scales"][..., None, None]
        _plain_bounds(s)
        return s["codes"] * s["scales"][..., None, None]
    if kind == "select":
        if not own:
            _plain_select(s)
        return [s["pages"], s["lens"]]
    if own:
        return s["out"]
    return _plain_selected(s) if kind == "selected" else _plain_shared(s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    hk, d, page = c["kv_heads"], c["dim"], c["page"]
    lens = _ints(c["lens"])
    if c["kind"] == "bounds":
        new = _ints(c["new"])
        rows = sum(n - (n - m) // page * page for n, m in zip(lens, new) if m)
        pages = sum(-(-n // page) - (n - m) // page for n, m in zip(lens, new) if m)
        return {"bytes": c["layers"] * hk * (rows * 2 * d + pages * (2 * d + 4)), "flops": c["layers"] * hk * rows * 2 * d}
    drafts, hq = _ints(c["drafts"]), c["q_heads"]
    tokens = sum(drafts)
    if c["kind"] == "select":
        between = [max(0, _spans(c, n, m)[1] - c["first"]) for n, m in zip(lens, drafts)]
        return {"bytes": hk * sum(between) * (2 * d + 8) + tokens * (2 * d * hq + hk * (4 * c["width"] + 8)), "flops": sum(b * m for b, m in zip(between, drafts)) * hq * 4 * d}
    if c["kind"] == "selected":
        read, seen = 0, 0
        for n, m in zip(lens, drafts):
            last, tail, k = _spans(c, n, m)
            between = max(0, tail - c["first"])
            ends = n + m - page * between
            # a quarter of the pages of each further token of a sequence are its own
            read += ends + page * min(between, k * (1 + (m - 1) / 4))
            seen += m * (ends - m + page * k) + m * (m + 1) // 2
        return {"bytes": 4 * d * (hq * tokens + hk * read) + 4 * tokens * hk * (c["width"] + 2), "flops": 4 * d * hq * seen}
    prefix = [p for p, n in zip(_ints(c["prefix"]), _ints(c["members"])) for _ in range(n)]
    keys = sum(_ints(c["prefix"])) + sum(lens) + tokens
    seen = sum((p + n) * m + m * (m + 1) // 2 for p, n, m in zip(prefix, lens, drafts))
    return {"bytes": 4 * d * (hq * tokens + hk * keys), "flops": 4 * d * hq * seen}


# ------------------------------------------------------------------------------------------------ 64 bits
def _softmax64(q, k, v, scale, seen):
    """One head's rows in 64 bits: q [rows, dim], k and v [keys, dim], seen [rows, keys]."""
    scores = torch.where(seen, (q @ k.T) * scale, -math.inf)
    return torch.nan_to_num(torch.softmax(scores, -1), nan=0.0) @ v


def _exponent(size):
    """The least e >= LEAST_EXPONENT with size <= 127 2^e, by trying."""
    e = torch.full_like(size, LEAST_EXPONENT)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):
        grown = e + step
        e = torch.where(size > 127 * torch.exp2(grown - 1), grown, e)
    return e


def exact(case, seed):
    """The definitions, sequence by sequence and head by head, in 64 bits."""
    c = case
    s = prepare(case, seed)
    hk, d, page = c["kv_heads"], c["dim"], c["page"]
    lens = _ints(c["lens"])
    if c["kind"] == "bounds":
        values = s["codes"].double() * s["scales"].double()[..., None, None]
        for i, (n, m) in enumerate(zip(lens, _ints(c["new"]))):
            for j in range((n - m) // page, -(-n // page)) if m else ():
                name = int(s["tables"][i, j])
                k = s["keys"][:, name, :, :min(page, n - j * page)].double()
                step = torch.exp2(_exponent(k.abs().amax((2, 3))))[..., None]
                values[:, name] = torch.stack((torch.ceil(k.max(2).values / step), torch.floor(k.min(2).values / step)), 2) * step[..., None]
        return values
    drafts, group = _ints(c["drafts"]), c["q_heads"] // hk
    starts = _offsets(drafts)
    if c["kind"] == "select":
        lists = [(m * hk, max(0, _spans(c, n, m)[1] - c["first"])) for n, m in zip(lens, drafts)]
        if sum(n for n, _ in lists) > 4000 or sum(n * b for n, b in lists) > 6e6:
            return None  # half a minute
        pages, out_lens = torch.full(s["pages"].shape, -1, dtype=torch.int32), torch.zeros(s["lens"].shape, dtype=torch.int32)
        for i, (n, m) in enumerate(zip(lens, drafts)):
            last, tail, k = _spans(c, n, m)
            first = min(c["first"], tail)
            names = s["tables"][i, first:tail].long()
            bounds = s["codes"][names].double() * s["scales"][names].double()[..., None, None]   # [pages, kv_heads, 2, dim]
            for t in range(m):
                q = s["q"][starts[i] + t].double()
                step = torch.exp2(_exponent(q.abs().amax(-1)))[:, None]
                q = (torch.round(q / step) * step).unflatten(0, (hk, group))
                for h in range(hk):
                    score = torch.maximum(q[h][:, None] * bounds[:, h, 0], q[h][:, None] * bounds[:, h, 1]).sum(-1).amax(0).cpu().tolist()
                    best = sorted(sorted(range(len(score)), key=lambda p: (-score[p], p))[:k])
                    which = list(range(first)) + [first + p for p in best] + list(range(tail, last))
                    pages[starts[i] + t, h, :len(which)] = s["tables"][i].cpu()[which]
                    held = n - page * (tail - first - k)
                    out_lens[starts[i] + t, h] = torch.tensor([held, held + (m if c["shape"] == "tree" else t + 1)])
        return [pages.cuda(), out_lens.cuda()]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    if c["kind"] == "selected":
        lens_of = s["lens"].tolist()
        for t in range(out.shape[0]):
            for h in range(hk):
                held, total = lens_of[t][h]
                names = s["pages"][t, h, :-(-total // page)].long()
                k, v = (x[names, h].flatten(0, 1)[:total].double() for x in (s["keys"], s["values"]))
                seen = torch.ones(1, total, device="cuda", dtype=torch.bool)
                if c["shape"] == "tree":
                    seen[0, held:] = (s["ancestors"][t] >> torch.arange(total - held, device="cuda")) & 1 == 1
                rows = slice(h * group, h * group + group)
                out[t, rows] = _softmax64(s["q"][t, rows].double(), k, v, s["scale"], seen)
        return out
    begins = [b for b, n in zip(_offsets(_ints(c["members"])), _ints(c["members"])) for _ in range(n)]
    prefix = [p for p, n in zip(_ints(c["prefix"]), _ints(c["members"])) for _ in range(n)]
    for i, (n, m) in enumerate(zip(lens, drafts)):
        total, rows = prefix[i] + n + m, slice(starts[i], starts[i + 1])
        names = torch.cat((s["tables"][begins[i], :prefix[i] // page], s["tables"][i, prefix[i] // page:-(-total // page)])).long()
        k, v = (x[names].transpose(1, 2).flatten(0, 1)[:total].double() for x in (s["keys"], s["values"]))
        seen = torch.ones(m, total, device="cuda", dtype=torch.bool)
        for j in range(m):
            seen[:, prefix[i] + n + j] = (s["ancestors"][rows] >> j) & 1 == 1
        for h in range(c["q_heads"]):
            out[rows, h] = _softmax64(s["q"][rows, h].double(), k[:, h // group], v[:, h // group], s["scale"], seen)
    return out
