"""Workloads of attention over a paged key/value cache: what a program that decodes with this framework's quantized projections does
between them.

`listed()` names twelve, `draw(rng)` makes more of the same ranges.  A case is one of these kinds:

  rope     q, k, v of some tokens from the projections (fp32 rows, or bf16 ones): rms_norm of every head of q and k (some models),
           rotation by position, rounding to bf16; q for the attention, k and v into the pages of the cache
  prompt   causal attention over whole prompts, packed one behind the other; keys and values packed too, or in the cache's pages, where a
           sequence may have a past that it attends to as well
  tree     attention of a few new tokens per sequence over a long cache: one token, a chain, or a tree of drafted tokens in which each
           sees the context and its own ancestors
  fork     pages copied to other pages in all layers, whole or the rows in use: sequences that go separate ways
  compact  the kept ones of the drafted tokens moved up to the end of the context in all layers

Lengths are texts, one number for each sequence.  A cache holds bf16 [layers, pages, kv_heads, page_tokens, dim]; token t of a
sequence lies in row t % page_tokens of page tables[sequence, t // page_tokens].
"""
from __future__ import annotations

import itertools
import math

import torch

own = False  # True: the framework's operators; False: the same from elementary operations

MAX_FLOPS = 1.1e12     # of a drawn prompt case, 4 * tokens^2 * heads * dim before the mask; the largest listed one has 1.1e12
MAX_CACHE = 600 << 20  # bytes of keys and values that a drawn tree case reads
EPS = 1e-5
DRAFTS = 64            # drafted tokens of a sequence, at most: a mask is one 64-bit word


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # One decoded token of the 7B-shape model: 32 heads, no norms, pairs (2i, 2i+1).  The smallest call.
        dict(name="rope_1tok", kind="rope", tokens=1, q_heads=32, kv_heads=32, dim=128, rot=128, x="f32", norm=False, pairs="adjacent", page=16, joined=False),
        # A 2048-token prompt of the 70B-shape model's heads, with norms of q and k.
        dict(name="rope_2048_norm", kind="rope", tokens=2048, q_heads=64, kv_heads=8, dim=128, rot=128, x="f32", norm=True, pairs="half", page=64, joined=False),
        # An odd number of bf16 rows out of one joined q|k|v buffer, heads of 96 of which 64 are rotated.
        dict(name="rope_777_bf16", kind="rope", tokens=777, q_heads=28, kv_heads=4, dim=96, rot=64, x="bf16", norm=True, pairs="half", page=32, joined=True),
        # A 512-token prompt of the 7B-shape model.
        dict(name="prompt_512", kind="prompt", lens="512", past="", q_heads=32, kv_heads=32, dim=128, page=0),
        # A long prompt, grouped heads: the largest call.
        dict(name="prompt_8192_gqa", kind="prompt", lens="8192", past="", q_heads=32, kv_heads=8, dim=128, page=0),
        # Prompts of several users in one call, some with a past in the cache, one empty.
        dict(name="prompt_ragged_pages", kind="prompt", lens="1000,37,1,0,513,1999,129,770", past="0,512,300,64,0,0,1023,41", q_heads=24, kv_heads=8, dim=64, page=16),
        # One token of the 7B-shape model at a context of 512.
        dict(name="decode_512", kind="tree", lens="512", drafts="1", shape="single", q_heads=32, kv_heads=32, dim=128, page=16),
        # A batch of sequences of the 70B-shape model's heads, one token each, contexts from 31 to 4000.
        dict(name="decode_batch", kind="tree", lens=",".join(str(31 + 61 * i + (i * i * 29) % 1200) for i in range(48)), drafts=",".join(["1"] * 48), shape="single",
             q_heads=64, kv_heads=8, dim=128, page=64),
        # Eight sequences with up to 24 drafted tokens in a tree.
        dict(name="tree_8seq", kind="tree", lens="1511,2040,903,2999,1,640,0,1777", drafts="24,24,17,24,5,24,24,1", shape="tree", q_heads=32, kv_heads=8, dim=128, page=32),
        # One sequence with a very long context and a chain of five drafted tokens.
        dict(name="chain_long", kind="tree", lens="131059", drafts="5", shape="chain", q_heads=64, kv_heads=8, dim=128, page=64),
        # Twenty-four sequences are forked: the page that each is writing is copied, as far as it is filled.
        dict(name="fork_24", kind="fork", layers=32, pairs=24, kv_heads=8, dim=128, page=64, partial=True),
        # After a step of drafting in sixteen sequences, the accepted tokens move up.
        dict(name="compact_16", kind="compact", layers=32, lens=",".join(str(100 + 77 * i) for i in range(16)), drafts=16, kv_heads=8, dim=128, page=64),
    ]


def _log(rng, lo, hi):
    return lo * (hi / lo) ** rng.random()


def _heads(rng):
    kv = rng.choice((1, 2, 4, 8, 8, 16, 32))
    group = rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 16) if kv * g <= 64])
    return kv * group, kv


def draw(rng):
    kind = rng.choice(("rope", "rope", "prompt", "prompt", "prompt", "tree", "tree", "tree", "tree", "fork", "compact"))
    q_heads, kv_heads = _heads(rng)
    dim = rng.choice((64, 64, 128, 128, 128, 80, 96, 112))
    page = rng.choice((16, 32, 64, 128))
    if kind == "rope":
        tokens = int(_log(rng, 1, 4096))
        rot = rng.choice((dim, dim, dim // 2))
        return dict(kind="rope", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, rot=rot, x=rng.choice(("f32", "f32", "bf16")),
                    norm=rng.random() < 0.6, pairs=rng.choice(("half", "half", "adjacent")), page=page, joined=rng.random() < 0.4)
    if kind == "prompt":
        most = int(math.sqrt(MAX_FLOPS / 4 / q_heads / dim) * 0.7)
        seqs = rng.choice((1, 1, rng.randint(2, 12)))
        total = min(most, 8192)
        lens = [max(1, int(_log(rng, 1, total / (1 if seqs == 1 else 4)))) for _ in range(seqs)]
        while sum(lens) > total:
            lens[lens.index(max(lens))] //= 2
        paged = rng.random() < 0.5
        past = [rng.choice((0, int(_log(rng, 1, 0.2 * total)))) for _ in lens] if paged else []
        while sum(past) > 0.3 * total:
            past[past.index(max(past))] //= 2
        return dict(kind="prompt", lens=",".join(map(str, lens)), past=",".join(map(str, past)), q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page if paged else 0)
    if kind == "tree":
        shape = rng.choice(("single", "single", "chain", "tree"))
        seqs = max(1, int(_log(rng, 1, 64)))
        per = kv_heads * dim * 4
        most = min(131072, MAX_CACHE // per // seqs)
        top = _log(rng, min(64, most), most)
        lens = [int(_log(rng, max(1, top / 8), top)) for _ in range(seqs)]
        drafts = [1 if shape == "single" else rng.randint(1, 8) if shape == "chain" else rng.randint(2, DRAFTS) for _ in range(seqs)]
        # the plain form's scores and gathered keys, padded to the longest, stay within a few GB
        while seqs * (max(lens) + max(drafts)) * (q_heads * max(drafts) * 4 + per) > 8 << 30:
            lens = [max(1, n // 2) for n in lens]
        return dict(kind="tree", lens=",".join(map(str, lens)), drafts=",".join(map(str, drafts)), shape=shape, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page)
    layers = rng.randint(1, 48)
    if kind == "fork":
        pairs = max(1, int(_log(rng, 1, 64)))
        while layers * pairs * kv_heads * page * dim * 8 > 1 << 30:
            pairs = (pairs + 1) // 2
            layers = (layers + 1) // 2
        return dict(kind="fork", layers=layers, pairs=pairs, kv_heads=kv_heads, dim=dim, page=page, partial=rng.random() < 0.7)
    seqs = max(1, int(_log(rng, 1, 48)))
    lens = [int(_log(rng, 1, 1500)) for _ in range(seqs)]
    while layers * (sum(lens) + seqs * (page + DRAFTS)) * kv_heads * dim * 4 > 2 << 30:
        lens, layers = [n // 2 for n in lens], (layers + 1) // 2
    return dict(kind="compact", layers=layers, lens=",".join(map(str, lens)), drafts=rng.randint(1, DRAFTS), kv_heads=kv_heads, dim=dim, page=page)


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


def prepare(case, seed):
    gen, c = _gen(seed), case
    host = torch.Generator().manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "rope":
        t, hq, hk, d, page = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
        kind = torch.float32 if c["x"] == "f32" else torch.bfloat16
        if c["joined"]:
            x = (torch.randn(t, (hq + 2 * hk) * d, device="cuda", generator=gen) * 1.5).to(kind)
            q, k, v = x[:, :hq * d], x[:, hq * d:(hq + hk) * d], x[:, (hq + hk) * d:]
        else:
            q, k, v = ((torch.randn(t, h * d, device="cuda", generator=gen) * 1.5).to(kind) for h in (hq, hk, hk))
        s.update(q=q.unflatten(1, (hq, d)), k=k.unflatten(1, (hk, d)), v=v.unflatten(1, (hk, d)))
        if c["norm"]:
            s.update(gamma_q=1 + 0.2 * torch.randn(d, device="cuda", generator=gen), gamma_k=1 + 0.2 * torch.randn(d, device="cuda", generator=gen))
        # the model's table of rotations, made once: (cos, sin) of position * 10000^(-2i / rot); the tokens lie somewhere in its range
        rows = max(8192, t + 100)
        angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        s["table"] = torch.stack((angle.cos(), angle.sin()), -1).float()
        first = int(torch.randint(0, rows - t + 1, (1,), generator=host))
        s["positions"] = torch.arange(first, first + t, device="cuda", dtype=torch.int32)
        pages = -(-t // page) + 2
        keys, values = (_normal(gen, pages, hk, page, d) for _ in range(2))
        order = torch.randperm(pages, device="cuda", generator=gen)
        at = torch.arange(t, device="cuda") + first % page
        s.update(keys=keys, values=values, slots=order[at // page] * page + at % page, q_out=torch.empty(t, hq, d, device="cuda", dtype=torch.bfloat16))
    elif c["kind"] == "prompt":
        lens, hq, hk, d = _ints(c["lens"]), c["q_heads"], c["kv_heads"], c["dim"]
        q = _normal(gen, sum(lens), hq, d, scale=1.5)
        s.update(q=q, q_offsets=_i32(_offsets(lens)), out=torch.empty_like(q), scale=1 / math.sqrt(d))
        if c["page"]:
            totals = [n + p for n, p in zip(lens, _ints(c["past"]))]
            s["tables"], pages = _pages(totals, c["page"], gen)
            s.update(keys=_normal(gen, pages, hk, c["page"], d), values=_normal(gen, pages, hk, c["page"], d), k_lens=_i32(totals))
        else:
            s.update(keys=_normal(gen, sum(lens), hk, d), values=_normal(gen, sum(lens), hk, d))
    elif c["kind"] == "tree":
        lens, drafts, hq, hk, d = _ints(c["lens"]), _ints(c["drafts"]), c["q_heads"], c["kv_heads"], c["dim"]
        q = _normal(gen, sum(drafts), hq, d, scale=1.5)
        s["tables"], pages = _pages([n + m for n, m in zip(lens, drafts)], c["page"], gen)
        s.update(q=q, out=torch.empty_like(q), keys=_normal(gen, pages, hk, c["page"], d), values=_normal(gen, pages, hk, c["page"], d), context=_i32(lens),
                 q_offsets=_i32(_offsets(drafts)), scale=1 / math.sqrt(d))
        s["ancestors"] = torch.tensor([w for n in drafts for w in _ancestors(n, c["shape"], host)], dtype=torch.int64, device="cuda")
    else:
        if c["kind"] == "fork":
            pages = 2 * c["pairs"] + 5
            order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
            s["pairs"] = torch.stack((order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]), 1).contiguous()
            s["rows"] = torch.randint(1, c["page"] + 1, (c["pairs"],), device="cuda", generator=gen, dtype=torch.int32) if c["partial"] else None
        else:
            lens, n = _ints(c["lens"]), c["drafts"]
            s["tables"], pages = _pages([m + n for m in lens], c["page"], gen)
            s["context"] = _i32(lens)
            # the kept drafts of each sequence, ascending, and how many they are
            pick = torch.rand(len(lens), n, device="cuda", generator=gen) < 0.4
            s["counts"] = pick.sum(1).to(torch.int32)
            s["kept"] = torch.where(pick, torch.arange(n, device="cuda"), n).sort(1).values.to(torch.int32)
        shape = (c["layers"], pages, c["kv_heads"], c["page"], c["dim"])
        s.update(keys=_normal(gen, *shape), values=_normal(gen, *shape))
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
    """A torch tensor's memory as the framework's tensor; tokens may lie further apart than they are long."""
    from warpforge_b200.backend import DeviceTensor

    names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.int32: "i32", torch.int64: "i64"}
    apart = t.stride(0) if t.dim() == 3 else 0
    return DeviceTensor(t.data_ptr(), tuple(t.shape), names[t.dtype], owner=t, row_stride=apart)


def _call(s):
    """The operator with its buffers bound, as a program keeps it for its loop."""
    from warpforge_b200 import attention

    c, ctx = s["case"], _context()
    h = {k: _held(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["kind"] == "rope":
        return attention.QkNormRope(ctx, h["q"], h["k"], h["v"], h["q_out"], h["keys"], h["values"], h["positions"], h["table"], slots=h["slots"], norm=c["norm"],
                                    gamma_q=h.get("gamma_q"), gamma_k=h.get("gamma_k"), eps=EPS, pairs=c["pairs"]).run
    if c["kind"] == "prompt":
        return attention.PromptAttention(ctx, h["q"], h["keys"], h["values"], h["out"], h["q_offsets"], tables=h.get("tables"), k_lens=h.get("k_lens"), scale=s["scale"]).run
    if c["kind"] == "tree":
        return attention.TreeAttention(ctx, h["q"], h["keys"], h["values"], h["out"], h["tables"], h["context"], max_context=max(_ints(c["lens"])), q_offsets=h["q_offsets"],
                                       max_drafts=max(_ints(c["drafts"])), ancestors=h["ancestors"], scale=s["scale"]).run
    cache = attention.KvCache(ctx, c["layers"], h["keys"].shape()[1], c["page"], c["kv_heads"], c["dim"], keys=h["keys"], values=h["values"])
    if c["kind"] == "fork":
        return lambda: cache.copy_pages(h["pairs"], h.get("rows"))
    return lambda: cache.compact(h["tables"], h["context"], h["kept"], h["counts"])


# ------------------------------------------------------------------------------------------------ their plain forms
def _rotated(x, c, table, positions):
    rot = c["rot"]
    cos, sin = (table[positions.long()][:, None, :, i] for i in (0, 1))
    if c["pairs"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _normed(x, gamma):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma


def _plain_rope(s):
    c = s["case"]
    q, k = s["q"].float(), s["k"].float()
    if c["norm"]:
        q, k = _normed(q, s["gamma_q"]), _normed(k, s["gamma_k"])
    at, row = s["slots"] // c["page"], s["slots"] % c["page"]
    s["keys"][at, :, row] = _rotated(k, c, s["table"], s["positions"]).bfloat16()
    s["values"][at, :, row] = s["v"].bfloat16()
    return [_rotated(q, c, s["table"], s["positions"]).bfloat16(), s["keys"], s["values"]]


def _weights(scores, seen):
    """Softmax over the keys that a row sees, in place; rows that see none get zeros."""
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(torch.where(total == 0, 1.0, total))


def _plain_prompt(s):
    c, q, k, v = s["case"], s["q"], s["keys"], s["values"]
    lens, hk = _ints(c["lens"]), c["kv_heads"]
    totals = [n + p for n, p in zip(lens, _ints(c["past"]))] if c["page"] else lens
    q_starts, k_starts = (torch.tensor(_offsets(n)[:-1], device="cuda") for n in (lens, totals))
    q_lens, k_lens = torch.tensor(lens, device="cuda"), torch.tensor(totals, device="cuda")
    rows, cols = torch.arange(sum(lens), device="cuda"), torch.arange(sum(totals), device="cuda")
    q_seq, k_seq = (torch.repeat_interleave(torch.arange(len(lens), device="cuda"), n, output_size=m) for n, m in ((q_lens, sum(lens)), (k_lens, sum(totals))))
    q_at, k_at = rows - q_starts[q_seq] + (k_lens - q_lens)[q_seq], cols - k_starts[k_seq]
    if c["page"]:
        page = s["tables"][k_seq, k_at // c["page"]].long()
        k, v = k[page, :, k_at % c["page"]], v[page, :, k_at % c["page"]]
    seen = (q_seq[:, None] == k_seq[None, :]) & (k_at[None, :] <= q_at[:, None])
    grouped = q.float().unflatten(1, (hk, -1)).permute(1, 2, 0, 3)  # [kv_heads, group, rows, dim]
    w = _weights(grouped @ k.float().permute(1, 2, 0)[:, None] * s["scale"], seen)
    return (w @ v.float().transpose(0, 1)[:, None]).permute(2, 0, 1, 3).flatten(1, 2).bfloat16()


def _plain_tree(s):
    c, q = s["case"], s["q"].float()
    lens, drafts, hk, page = _ints(c["lens"]), _ints(c["drafts"]), c["kv_heads"], c["page"]
    most, widest = max(n + m for n, m in zip(lens, drafts)), max(drafts)
    at = torch.arange(most, device="cuda")
    where = s["tables"][:, (at // page).clamp(max=s["tables"].shape[1] - 1)].long()          # [seqs, keys]
    k, v = (x[where, :, at % page].float().transpose(1, 2) for x in (s["keys"], s["values"]))  # [seqs, kv_heads, keys, dim]
    start = s["q_offsets"][:-1].long()
    count = s["q_offsets"][1:].long() - start
    row = (start[:, None] + torch.arange(widest, device="cuda")[None, :]).clamp(max=q.shape[0] - 1)
    queries = q[row].unflatten(2, (hk, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)               # [seqs, kv_heads, group * drafts, dim]
    draft = at[None, :] - s["context"].long()[:, None]                                         # [seqs, keys]
    bit = (s["ancestors"][row][:, :, None] >> draft.clamp(0, 63)[:, None, :]) & 1
    seen = (draft[:, None, :] < 0) | ((draft[:, None, :] < count[:, None, None]) & (draft[:, None, :] < DRAFTS) & (bit == 1))  # [seqs, drafts, keys]
    w = _weights(queries @ k.transpose(2, 3) * s["scale"], seen[:, None].repeat(1, 1, q.shape[1] // hk, 1))
    out = (w @ v).unflatten(2, (-1, widest)).permute(0, 3, 1, 2, 4).flatten(2, 3)              # [seqs, drafts, heads, dim]
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), count, output_size=q.shape[0])
    return out[seq, torch.arange(q.shape[0], device="cuda") - start[seq]].bfloat16()


def _plain_pages(s):
    c, page = s["case"], s["case"]["page"]
    if c["kind"] == "fork":
        src, dst = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
        filled = s["rows"] if s["rows"] is not None else torch.full_like(s["pairs"][:, 0], page)
        taken = (torch.arange(page, device="cuda")[None, :] < filled[:, None])[None, :, None, :, None]
        s["keys"][:, dst] = torch.where(taken, s["keys"][:, src], s["keys"][:, dst])
        s["values"][:, dst] = torch.where(taken, s["values"][:, src], s["values"][:, dst])
    else:
        i = torch.arange(c["drafts"], device="cuda")[None, :]
        to = s["context"].long()[:, None] + i
        come = torch.where(i < s["counts"][:, None], s["context"].long()[:, None] + s["kept"], to)
        (p, r), (n, m) = ((torch.gather(s["tables"].long(), 1, a // page), a % page) for a in (come, to))
        s["keys"][:, n, :, m] = s["keys"][:, p, :, r]
        s["values"][:, n, :, m] = s["values"][:, p, :, r]


def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        if "call" not in s:
            s["call"] = _call(s)
        s["call"]()
    if kind == "rope":
        return [s["q_out"], s["keys"], s["values"]] if own else _plain_rope(s)
    if kind == "prompt":
        return s["out"] if own else _plain_prompt(s)
    if kind == "tree":
        return s["out"] if own else _plain_tree(s)
    if not own:
        _plain_pages(s)
    return [s["keys"].view(torch.int16), s["values"].view(torch.int16)]  # bits: a copy is a copy


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    hk, d = c["kv_heads"], c["dim"]
    if c["kind"] == "rope":
        t, hq = c["tokens"], c["q_heads"]
        size = 4 if c["x"] == "f32" else 2
        # q, k, v in, q, k, v out in bf16, a row of the table, a position and a slot for each token
        return {"bytes": t * ((hq + 2 * hk) * d * (size + 2) + c["rot"] * 4 + 12), "flops": t * (hq + hk) * (3 * c["rot"] + (4 * d if c["norm"] else 0))}
    if c["kind"] == "prompt":
        lens, hq = _ints(c["lens"]), c["q_heads"]
        past = _ints(c["past"]) if c["page"] else [0] * len(lens)
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lens, past))
        return {"bytes": 2 * d * (2 * hq * sum(lens) + 2 * hk * (sum(lens) + sum(past))), "flops": 4 * d * hq * pairs}
    if c["kind"] == "tree":
        lens, drafts, hq = _ints(c["lens"]), _ints(c["drafts"]), c["q_heads"]
        keys = sum(lens) + sum(drafts)
        seen = sum(n * m + m * (m + 1) // 2 for n, m in zip(lens, drafts))
        return {"bytes": 2 * d * (2 * hq * sum(drafts) + 2 * hk * keys) + 8 * sum(drafts), "flops": 4 * d * hq * seen}
    if c["kind"] == "fork":
        rows = c["pairs"] * (c["page"] + 1) / 2 if c["partial"] else c["pairs"] * c["page"]
        return {"bytes": c["layers"] * rows * hk * d * 8, "flops": 0}
    return {"bytes": c["layers"] * len(_ints(c["lens"])) * 0.4 * c["drafts"] * hk * d * 8, "flops": 0}


# ------------------------------------------------------------------------------------------------ 64 bits
def _softmax64(q, k, v, scale, seen):
    """One head's rows in 64 bits: q [rows, dim], k and v [keys, dim], seen [rows, keys]."""
    scores = torch.where(seen, (q @ k.T) * scale, -math.inf)
    p = torch.nan_to_num(torch.softmax(scores, -1), nan=0.0)
    return p @ v


def exact(case, seed):
    """The definition, sequence by sequence and head by head, in 64 bits; copies of pages have no computed numbers."""
    c = case
    if c["kind"] in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    hk, d = c["kv_heads"], c["dim"]
    if c["kind"] == "rope":
        turn = torch.view_as_complex(s["table"].double()[s["positions"].long()])[:, None]
        done = []
        for x, gamma in ((s["q"].double(), s.get("gamma_q")), (s["k"].double(), s.get("gamma_k"))):
            if c["norm"]:
                x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * gamma.double()
            half = c["rot"] // 2
            first = torch.arange(half, device="cuda") * (1 if c["pairs"] == "half" else 2)
            second = first + (half if c["pairs"] == "half" else 1)
            pair = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = pair.real, pair.imag
            done.append(y)
        keys, values = s["keys"].double(), s["values"].double()
        for t, slot in enumerate(s["slots"].tolist()):
            keys[slot // c["page"], :, slot % c["page"]] = done[1][t]
            values[slot // c["page"], :, slot % c["page"]] = s["v"][t].double()
        return [done[0], keys, values]
    group = c["q_heads"] // hk
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    lens = _ints(c["lens"])
    if c["kind"] == "prompt":
        news, olds = lens, _ints(c["past"]) if c["page"] else [0] * len(lens)
    else:
        news, olds = _ints(c["drafts"]), lens
    starts = _offsets(news)
    for i, (new, old) in enumerate(zip(news, olds)):
        if not new:
            continue
        total, rows = new + old, slice(starts[i], starts[i + 1])
        if c["page"]:
            names = s["tables"][i, :-(-total // c["page"])].long()
            k, v = (x[names].transpose(1, 2).flatten(0, 1)[:total].double() for x in (s["keys"], s["values"]))
        else:
            k, v = s["keys"][rows].double(), s["values"][rows].double()
        seen = torch.ones(new, total, device="cuda", dtype=torch.bool)
        if c["kind"] == "prompt":
            seen = seen.tril(old)
        else:
            words = s["ancestors"][rows]
            for j in range(new):
                seen[:, old + j] = (words >> j) & 1 == 1
        for h in range(c["q_heads"]):
            out[rows, h] = _softmax64(s["q"][rows, h].double(), k[:, h // group], v[:, h // group], s["scale"], seen)
    return out
