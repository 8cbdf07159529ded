"""Operators of a decoder's batch over the paged cache: what they are measured on.

Beside the layer's own operators a serving program needs, for the sequences that it runs together:

* ``rope``  -- ``rope``: queries and keys turned by their positions' angles; halves or pairs, a part of the head, angles
  of far positions, frequencies scaled for long contexts.
* ``pages`` -- ``pages_trim`` and ``pages_grow``: tokens taken back (all of a finished sequence's, or rejected drafts),
  pages handed out for the new ones, and for every new row its position and its slot in the cache.
* ``beam``  -- ``beam_step``: the best continuations of every group of beams, with their histories in their new order.
* ``fork``  -- ``pages_fork``, ``pages_grow`` and ``kv_copy``: beams take over each other's pages; the last one, where it is
  shared, is copied before it is written.
* ``kv4``   -- ``kv_append`` and ``kv_read`` on a cache of 4 bits a value.
* ``attn4`` -- ``attn`` over such a cache, one new token a sequence or many.

Four bits hold a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; 32 dims of a row share a scale, the smallest power of two
with which the largest of them is at most 6 (stored as its exponent + 127). A byte holds two dims. Keys lie as
[page][head][position][dim / 2], values as [page][head][dim / 2][position], scales as [page][head][dim / 32][position].
A value that lies between two codes goes to the nearer one, halfway to the one whose number is even.

The free pages with the lowest numbers are handed out first, to the sequences in order. Equal totals of beams go to
the lowest (beam, token).
"""
import math
import os
import sys

import torch

own = False

STOP = 3   # the beams' stop token


def listed():
    return [
        # A batch's AR step: one row a sequence, heads turned whole.
        {"name": "rope_64", "kind": "rope", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 50, "past_hi": 1500,
         "heads": 20, "kv_heads": 20, "dim": 64, "rot": 64, "layout": "half", "dtype": "bf16", "scaling": "none"},
        # Prompts of a text model with shared heads, half of each head turned, behind a long document.
        {"name": "rope_prompts", "kind": "rope", "seqs": 9, "new_lo": 301, "new_hi": 2403, "past_lo": 0,
         "past_hi": 120000, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64, "layout": "pairs", "dtype": "bf16",
         "scaling": "parts"},
        # A batch's AR step with drafts: up to four tokens come, as many were taken back.
        {"name": "pages_64", "kind": "pages", "seqs": 64, "new_lo": 1, "new_hi": 4, "past_lo": 50, "past_hi": 1500,
         "page": 16, "spare": 1.5, "prompts": False},
        # A large server: a third of the sequences end and others come in with their prompts, one token for the rest.
        {"name": "pages_prompts", "kind": "pages", "seqs": 1000, "new_lo": 70, "new_hi": 1500, "past_lo": 100,
         "past_hi": 1900, "page": 16, "spare": 1.3, "prompts": True},
        # A batch of utterances, four beams each, the semantic vocabulary, the pipeline's penalty and temperature.
        {"name": "beam_64", "kind": "beam", "groups": 64, "width": 4, "vocab": 8194, "dtype": "f32", "temp": 0.8,
         "pen": 10.0, "hist": 1500},
        # Few utterances of a text model's vocabulary, wide beams.
        {"name": "beam_vocab", "kind": "beam", "groups": 24, "width": 8, "vocab": 151936, "dtype": "bf16",
         "temp": 1.0, "pen": 1.0, "hist": 600},
        # The beams' caches in their new order: two layers of the utterances' decoder.
        {"name": "fork_64", "kind": "fork", "groups": 64, "width": 4, "past_lo": 50, "past_hi": 1500, "layers": 2,
         "heads": 20, "dim": 64, "page": 16, "store": "q4"},
        # A batch's AR step: one token a row.
        {"name": "kv4_64", "kind": "kv4", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 50, "past_hi": 900,
         "heads": 20, "dim": 64, "page": 16, "back": "new"},
        # Prompts behind a prefix that the cache holds already; whole sequences go out to another worker.
        {"name": "kv4_prompts", "kind": "kv4", "seqs": 24, "new_lo": 70, "new_hi": 1500, "past_lo": 0,
         "past_hi": 333, "heads": 20, "dim": 64, "page": 64, "back": "all"},
        # A batch's AR step, every row of its own length.
        {"name": "attn4_64", "kind": "attn4", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 50, "past_hi": 1500,
         "heads": 20, "kv_heads": 20, "dim": 64, "page": 16, "left": False},
        # Few long rows of a text model with shared heads.
        {"name": "attn4_6_long", "kind": "attn4", "seqs": 6, "new_lo": 1, "new_hi": 1, "past_lo": 12000,
         "past_hi": 50001, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "left": False},
        # Prompts of a batch, some behind a prefix, some padded on the left.
        {"name": "attn4_prompts", "kind": "attn4", "seqs": 12, "new_lo": 500, "new_hi": 2100, "past_lo": 0,
         "past_hi": 300, "heads": 20, "kv_heads": 20, "dim": 64, "page": 16, "left": True},
    ]


def _log(rng, lo, hi, unit=1):
    """A multiple of `unit` from lo to hi (themselves multiples), uniform in its logarithm."""
    n = unit * int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / unit))
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(["rope", "rope", "pages", "beam", "beam", "fork", "kv4", "attn4", "attn4", "attn4"])
    if kind == "rope":
        heads, kv_heads, dim = rng.choice([(20, 20, 64), (32, 8, 128), (16, 2, 64), (10, 5, 256), (12, 12, 80)])
        rot = rng.choice([dim, dim // 2, dim // 4])
        new = rng.choice([1, _log(rng, 1, 2400)])
        most = 9 * 1350 * 40 * 128 // ((heads + kv_heads) * dim * new * 2)
        return {"kind": kind, "seqs": max(1, min(_log(rng, 1, 256), most)), "new_lo": max(1, new // 8), "new_hi": new,
                "past_lo": 0, "past_hi": _log(rng, 1, 400000), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rot, "layout": rng.choice(["half", "pairs"]), "dtype": rng.choice(["bf16", "bf16", "f32"]),
                "scaling": rng.choice(["none", "linear", "parts"])}
    if kind == "pages":
        prompts, new = rng.random() < 0.5, rng.choice([1, rng.randint(2, 8)])
        if prompts:
            new = _log(rng, 16, 1500)
        return {"kind": kind, "seqs": _log(rng, 1, 1000), "new_lo": max(1, new // 8), "new_hi": new, "past_lo": 1,
                "past_hi": _log(rng, 2, 1900), "page": rng.choice([16, 32, 64, 128]),
                "spare": rng.choice([1.1, 1.5, 4.0]), "prompts": prompts}
    if kind == "beam":
        vocab = rng.choice([8194, _log(rng, 100, 20000), _log(rng, 20000, 151936)])
        width = rng.choice([1, 2, 3, 4, 5, 8, 16])
        groups = max(1, min(_log(rng, 1, 128), 24 * 8 * 151936 // (width * vocab)))
        return {"kind": kind, "groups": groups, "width": width, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]),
                "temp": rng.choice([1.0, 0.8]), "pen": rng.choice([1.0, 10.0, 1.3]), "hist": _log(rng, 1, 1500)}
    if kind == "fork":
        width = rng.choice([2, 3, 4, 8])
        heads, dim = rng.choice([(20, 64), (8, 128), (5, 256)])
        past = _log(rng, 2, 1500)
        groups = max(1, min(_log(rng, 1, 64), 64 * 4 * 800 // (width * past)))
        return {"kind": kind, "groups": groups, "width": width, "past_lo": max(1, past // 8), "past_hi": past,
                "layers": rng.randint(1, 3), "heads": heads, "dim": dim, "page": rng.choice([16, 32, 64]),
                "store": rng.choice(["bf16", "q8", "q4"])}
    heads, kv_heads, dim = rng.choice([(20, 20, 64), (20, 20, 64), (16, 4, 128), (32, 8, 128), (16, 2, 64),
                                       (12, 12, 96), (10, 5, 256)])
    page = rng.choice([16, 32, 64, 128])
    if kind == "kv4":
        new, past = _log(rng, 1, 1500), _log(rng, 1, 1500)
        seqs = max(1, min(_log(rng, 1, 128), 24 * 950 * 20 * 64 // ((new + past) * kv_heads * dim)))
        return {"kind": kind, "seqs": seqs, "new_lo": max(1, new // 8), "new_hi": new, "past_lo": past // 8,
                "past_hi": past, "heads": kv_heads, "dim": dim, "page": page, "back": rng.choice(["new", "all"])}
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "left": rng.random() < 0.3}
    if rng.random() < 0.6:   # single tokens, or a few that are checked together
        new = rng.choice([1, 1, 1, rng.randint(2, 8)])
        past = _log(rng, 1, 50000)
        most = 6 * 31000 * 8 * 128 // (kv_heads * dim * (past + new))
        return {**c, "seqs": max(1, min(_log(rng, 1, 256), most)), "new_lo": 1, "new_hi": new, "past_lo": past // 4,
                "past_hi": past}
    new, past = _log(rng, 16, 2100), _log(rng, 1, 2000)
    most = 12 * 20 * 64 * 2100 * 2400 // (heads * dim * new * (new + past))
    return {**c, "seqs": max(1, min(_log(rng, 1, 32), most)), "new_lo": max(1, new // 4), "new_hi": new, "past_lo": 0,
            "past_hi": past}


def _spread(lo, hi, n):
    """n whole numbers between lo and hi, both among them where n allows, in no order."""
    if n == 1:
        return [hi]
    at = sorted(range(n), key=lambda i: math.fmod(0.6180339887498949 * (i + 1), 1.0))
    return [lo + (hi - lo) * i // (n - 1) for i in at]


def _lengths(case):
    """Of every sequence: its new tokens, and all its tokens."""
    new = _spread(case["new_lo"], case["new_hi"], case["seqs"])
    past = _spread(case["past_lo"], case["past_hi"], case["seqs"])[::-1]
    return new, [n + p for n, p in zip(new, past)]


def _moves(case):
    """pages: of every sequence its tokens before the pass, and how many leave and come."""
    new = _spread(case["new_lo"], case["new_hi"], case["seqs"])
    past = _spread(case["past_lo"], case["past_hi"], case["seqs"])[::-1]
    if not case["prompts"]:
        return [n + p for n, p in zip(new, past)], new, new
    ends = [b % 3 == 1 or len(new) == 1 for b in range(len(new))]
    had = [n if e else p for n, p, e in zip(new, past, ends)]
    return had, [n if e else 1 for n, e in zip(had, ends)], [n if e else 1 for n, e in zip(had, ends)]


def _firsts(case, lens):
    """The first position that a sequence's tokens see: behind the padding, for every third sequence."""
    return [(n // 3 if b % 3 == 0 else 0) if case["left"] else 0 for b, n in enumerate(lens)]


# ---- inputs ----------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    return _ints([0] + torch.tensor(counts).cumsum(0).tolist())


def _frequencies(rot, scaling):
    """Radians a position, 64 bits: as a text model has them, its positions eight times as dense, or so only where a
    turn takes more than a quarter of the 8192 positions that it was trained with, blended in between."""
    f = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        f = f / 8.0
    if scaling == "parts":
        turns = 8192.0 * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / 3.0).clamp(0.0, 1.0)
        f = f * keep + f / 8.0 * (1.0 - keep)
    return f.cuda()


def _channels(g, heads, dim):
    """Sizes of keys' and values' channels: a few are much larger than the others."""
    size = torch.exp(0.4 * _randn(g, heads, dim))
    return torch.where(torch.rand((heads, dim), generator=g, device="cuda") < 0.02, 6.0 * size, size)


def _table(g, need, n_pages, width):
    """Block table of sequences with these numbers of pages, handed out in no order; -1 behind the last."""
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    need = torch.tensor(need, device="cuda")
    at = torch.arange(width, device="cuda")
    index = (need.cumsum(0) - need)[:, None] + at
    return torch.where(at < need[:, None], order[index.clamp_max(n_pages - 1)], -1).contiguous()


def _free_bits(refs):
    """Bit p % 32 of word p / 32: page p is free."""
    pad = torch.zeros(-len(refs) % 32, dtype=torch.int64, device="cuda")
    free = torch.cat([(refs == 0).long(), pad]).view(-1, 32)
    word = (free << torch.arange(32, device="cuda")).sum(dim=1)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)


def _nibbles(codes):
    """Codes of two neighbours of the last dimension in a byte."""
    return (codes[..., 0::2] | codes[..., 1::2] << 4).contiguous()


def _cache4(case, g, lens, heads):
    """A paged cache of 4 bits with every page written before: pages, scales, and each sequence's pages."""
    page, dim = case["page"], case["dim"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    c = {"table": _table(g, need, pages, max(need))}
    for name in ("k", "v"):
        x = (_randn(g, pages, heads, page, dim) * _channels(g, heads, dim)[:, None]).to(torch.bfloat16)
        code, e = _codes4(x.float())
        code = _nibbles(code)
        c[name] = code if name == "k" else code.transpose(2, 3).contiguous()
        c[name + "_scale"] = e.transpose(2, 3).contiguous()
    return c


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = dict(case)
    if kind == "rope":
        new, lens = _lengths(case)
        t, heads, kv = torch.float32 if case["dtype"] == "f32" else torch.bfloat16, case["heads"], case["kv_heads"]
        # as a layer's product gives them: queries, keys and values side by side
        qkv = _randn(g, sum(new), heads + 2 * kv, case["dim"]).to(t)
        s["q"], s["k"] = qkv[:, :heads], qkv[:, heads:heads + kv]
        s["q_out"], s["k_out"] = (torch.empty(x.shape, dtype=t, device="cuda") for x in (s["q"], s["k"]))
        s["lens"], s["off"] = _ints(lens), None if max(new) == 1 else _offsets(new)
        s["freq"] = _frequencies(case["rot"], case["scaling"])
        s["factor"] = 1.0 if case["scaling"] == "none" else 1.1
    elif kind == "pages":
        had, drop, new = _moves(case)
        page = case["page"]
        need = [-(-n // page) for n in had]
        pages = int(sum(need) * case["spare"]) + 64
        s["table"] = _table(g, need, pages, max(need) + 1)
        # half of the others are held too, by prompts' beginnings that are kept
        s["refs"] = (torch.rand(pages, generator=g, device="cuda") < 0.5).to(torch.int32)
        s["refs"][s["table"][s["table"] >= 0].long()] = 1
        s["free"], s["lens"], s["missing"] = _free_bits(s["refs"]), _ints(had), _ints([0])
        s["drop"], s["new"] = _ints(drop), None if max(new) == 1 else _ints(new)
        s["off"] = torch.empty(len(had) + 1, dtype=torch.int32, device="cuda")
        s["pos"], s["slot"] = (torch.empty(sum(new), dtype=torch.int32, device="cuda") for _ in "ps")
    elif kind == "beam":
        rows, vocab, width = case["groups"] * case["width"], case["vocab"], case["width"]
        s["logits"] = _randn(g, rows, vocab).mul_(3.0).to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
        s["score"] = _randn(g, rows).mul_(0.7).sub_(20.0)
        s["done"] = (torch.rand(rows, generator=g, device="cuda") < 0.1).to(torch.uint8)
        s["temp_rows"] = None if case["temp"] == 1.0 else torch.full((rows,), case["temp"], device="cuda")
        s["pen_rows"] = None if case["pen"] == 1.0 else torch.full((rows,), case["pen"], device="cuda")
        words = -(-vocab // 32)
        # a twentieth of the vocabulary has come; places behind the last token are never set
        odds = torch.rand((rows, words * 32), generator=g, device="cuda") < 0.05
        odds[:, vocab:] = False
        s["bits"] = -_free_bits(odds.reshape(-1).to(torch.int32)).view(rows, words) - 1
        s["tokens"] = torch.randint(0, vocab, (rows, case["hist"]), generator=g, device="cuda").to(torch.int32)
        s["bits_out"], s["tokens_out"] = torch.empty_like(s["bits"]), torch.empty_like(s["tokens"])
        s["score_out"], s["done_out"] = torch.empty_like(s["score"]), torch.empty_like(s["done"])
        s["parent"], s["token"] = (torch.empty(rows, dtype=torch.int32, device="cuda") for _ in "pt")
    elif kind == "fork":
        page, width, groups, heads, dim = case["page"], case["width"], case["groups"], case["heads"], case["dim"]
        lens = [n + 1 for n in _spread(case["past_lo"], case["past_hi"], groups) for _ in range(width)]
        # the beams of a group share all pages but the last two
        need = [-(-n // page) for n in lens]
        pages = sum(need) * 2 + 3
        table = _table(g, need, pages, max(need) + 1)
        shared = torch.arange(table.shape[1], device="cuda") < torch.tensor(need, device="cuda")[:, None] - 2
        first = table.view(groups, width, -1)[:, :1].expand(-1, width, -1).reshape(table.shape)
        s["table"] = torch.where(shared, first, table).contiguous()
        held = s["table"][s["table"] >= 0].long()
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda").index_add_(
            0, held, torch.ones(len(held), dtype=torch.int32, device="cuda"))
        s["free"], s["lens"], s["missing"] = _free_bits(s["refs"]), _ints(lens), _ints([0])
        s["parent"] = torch.randint(0, width, (groups * width,), generator=g, device="cuda").to(torch.int32)
        s["ones"] = torch.ones(groups * width, dtype=torch.int32, device="cuda")
        s["copies"] = torch.empty((groups * width, 2), dtype=torch.int32, device="cuda")
        s["caches"] = []
        for _ in range(case["layers"]):
            c = {"table": s["table"]}
            for name in ("k", "v"):
                c[name], c[name + "_scale"] = _pool(g, case["store"], name, pages, heads, page, dim)
            s["caches"].append(c)
    else:
        new, lens = _lengths(case)
        total, heads, dim = sum(new), case.get("kv_heads", case["heads"]), case["dim"]
        s.update(_cache4(case, g, lens, heads))
        s["lens"], s["off"], s["max_new"] = _ints(lens), None if max(new) == 1 else _offsets(new), max(new)
        if kind == "kv4":
            # as a layer's product gives them: queries, keys and values side by side
            qkv = (_randn(g, total, 3, heads, dim) * _channels(g, heads, dim)).to(torch.bfloat16)
            s["k_new"], s["v_new"] = qkv[:, 1], qkv[:, 2]
            s["back_off"] = s["off"] if case["back"] == "new" else _offsets(lens)
            n = total if case["back"] == "new" else sum(lens)
            s["k_out"], s["v_out"] = (torch.empty((n, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in "kv")
        else:
            s["q"] = _randn(g, total, case["heads"], dim).to(torch.bfloat16)
            s["first"] = _ints(_firsts(case, lens)) if case["left"] else None
            s["out"] = torch.empty_like(s["q"])
    if own:   # the handles that a serving program holds
        p = _package()
        if kind in ("pages", "fork"):
            s["handle"] = p.Pages(s["table"], s["lens"], s["refs"], s["free"], case["page"], s["missing"])
        if kind == "fork":
            s["kv"] = [p.KvCache(c["k"], c["v"], c["table"], c["k_scale"], c["v_scale"]) for c in s["caches"]]
        if kind in ("kv4", "attn4"):
            s["cache"] = p.KvCache(s["k"], s["v"], s["table"], s["k_scale"], s["v_scale"])
    return s


def _pool(g, store, name, pages, heads, page, dim):
    """One tensor of a layer's cache and its scales, filled as earlier sequences left it."""
    if store == "bf16":
        shape = (pages, heads, page, dim) if name == "k" else (pages, heads, dim, page)
        return _randn(g, *shape).to(torch.bfloat16), None
    if store == "q8":
        shape = (pages, heads, page, dim) if name == "k" else (pages, heads, dim, page)
        return (torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8),
                torch.rand((pages, heads, page), generator=g, device="cuda"))
    shape = (pages, heads, page, dim // 2) if name == "k" else (pages, heads, dim // 2, page)
    return (torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(120, 130, (pages, heads, dim // 32, page), generator=g, device="cuda", dtype=torch.uint8))


# ---- one pass, plain -----------------------------------------------------------------

def _power(e):
    """2^e, for whole e from -126 to 127; below them 2^-126, which only blocks of zeros have."""
    return (e.clamp_min(-126) + 127 << 23).view(torch.float32)


def _codes4(x):
    """4-bit codes of rows of the last dimension, and their blocks' exponents + 127."""
    block = x.unflatten(-1, (-1, 32))
    top = block.abs().amax(dim=-1)
    m, e = torch.frexp(top)                        # top = m 2^e, m from 0.5 to 1: below or at 6 2^(e - 3) up to 0.75
    e = torch.where(m > 0.75, e - 2, e - 3).clamp(-127, 127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    y = (block / _power(e)[..., None]).flatten(-2)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return (code + 8 * (y < 0)).to(torch.uint8), (e + 127).to(torch.uint8)


def _values4(code, e):
    """The values of unpacked codes [..., dim] with exponents + 127 of their blocks [..., dim / 32]."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    x = torch.cat([grid, -grid])[code.int()]
    return (x.unflatten(-1, (-1, 32)) * _power(e.int() - 127)[..., None]).flatten(-2)


def _positions(s, off):
    """Of every row of the packed tensors with these offsets: its sequence and its position."""
    lens = s["lens"].long()
    off = torch.arange(len(lens) + 1, device="cuda") if off is None else off.long()
    n = off[1:] - off[:-1]
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), n)
    return seq, lens[seq] - n[seq] + torch.arange(len(seq), device="cuda") - off[seq]


def _plain_rope(s):
    angle = _positions(s, s["off"])[1].double()[:, None] * s["freq"]
    cos, sin = (f(angle).float()[:, None] * s["factor"] for f in (torch.cos, torch.sin))
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        turn, rest = x[..., :s["rot"]], x[..., s["rot"]:]
        if s["layout"] == "half":
            a, b = turn[..., :s["rot"] // 2], turn[..., s["rot"] // 2:]
            turn = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        else:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
        out[name] = torch.cat([turn, rest], dim=-1).to(s[name].dtype)
    return out


def _bits_of(words, n):
    """The first n bits of rows of 32-bit words."""
    return (words[..., None] >> torch.arange(32, device="cuda") & 1).flatten(-2)[..., :n]


def _set_free(s, page, value):
    free = _bits_of(s["free"], len(s["refs"]))
    free[page] = value
    s["free"].copy_(_free_bits(1 - free))


def _plain_trim(s, drop):
    page, table, lens = s["page"], s["table"], s["lens"]
    left = (lens - drop).clamp_min(0)
    at = torch.arange(table.shape[1], device="cuda")
    gone = (at >= ((left + page - 1) // page)[:, None]) & (table >= 0)
    held = table[gone].long()
    s["refs"].index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    table.masked_fill_(gone, -1)
    _set_free(s, held[s["refs"][held] == 0], 1)
    lens.copy_(left)


def _plain_grow(s, new, copies=None):
    """New pages for new[b] more tokens; where copies is given, shared last pages are replaced first."""
    page, table, lens, refs = s["page"], s["table"], s["lens"], s["refs"]
    seq = torch.arange(len(lens), device="cuda")
    before, after = (lens + page - 1) // page, (lens + new + page - 1) // page
    swap = torch.zeros_like(lens, dtype=torch.bool)
    if copies is not None:
        copies.fill_(-1)
        last = table.gather(1, (before - 1).clamp_min(0).long()[:, None])[:, 0].long()
        part = (lens % page > 0) & (new > 0) & (last >= 0)
        swap = part & (refs[last.clamp_min(0)] > 1)
        users = torch.zeros_like(refs).index_add_(0, last[swap], torch.ones_like(refs[last[swap]]))
        # of the sequences that hold a page, if all of them go on, the last one keeps it
        keeps = torch.full_like(refs, -1).scatter_reduce_(0, last[swap], seq[swap].int(), "amax")
        swap = swap & ~((users == refs)[last.clamp_min(0)] & (keeps[last.clamp_min(0)] == seq))
        refs.index_add_(0, last[swap], torch.full_like(refs[last[swap]], -1))
        copies[swap, 0] = last[swap].int()
    need = (after - before + swap).long()
    row = torch.repeat_interleave(seq, need)
    nth = torch.arange(len(row), device="cuda") - (need.cumsum(0) - need)[row]
    at = before.long()[row] - swap.long()[row] + nth
    got = torch.nonzero(_bits_of(s["free"], len(refs)))[:, 0][:len(row)]   # there are enough
    table[row, at] = got.int()
    refs[got] = 1
    _set_free(s, got, 0)
    if copies is not None:
        copies[row[swap[row] & (nth == 0)], 1] = got[swap[row] & (nth == 0)].int()
    lens.add_(new)


def _plain_pages(s):
    new = torch.ones_like(s["lens"]) if s["new"] is None else s["new"]
    _plain_trim(s, s["drop"])
    _plain_grow(s, new)
    s["off"][0] = 0
    s["off"][1:] = new.cumsum(0)
    seq, pos = _positions(s, s["off"])
    s["pos"].copy_(pos)
    s["slot"].copy_(s["table"][seq, pos // s["page"]] * s["page"] + pos % s["page"])
    return {n: s[n] for n in ("table", "lens", "refs", "free", "off", "pos", "slot", "missing")}


def _plain_fork(s):
    width = s["width"]
    _plain_trim(s, s["ones"])
    rows = torch.arange(len(s["parent"]), device="cuda")
    source = rows // width * width + s["parent"].long()
    held = s["table"][s["table"] >= 0].long()
    s["refs"].index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    s["table"].copy_(s["table"][source])
    s["lens"].copy_(s["lens"][source])
    now = s["table"][s["table"] >= 0].long()
    s["refs"].index_add_(0, now, torch.ones_like(now, dtype=torch.int32))
    _set_free(s, held[s["refs"][held] == 0], 1)
    _plain_grow(s, s["ones"], s["copies"])
    out = {n: s[n] for n in ("table", "lens", "refs", "free", "copies", "missing")}
    src, dst = s["copies"][s["copies"][:, 1] >= 0].long().unbind(1)
    for i, c in enumerate(s["caches"]):
        for name in ("k", "v", "k_scale", "v_scale"):
            if c[name] is not None:
                c[name][dst] = c[name][src]
                out["%s%d" % (name, i)] = c[name]
    return out


def _plain_beam(s):
    rows, width, vocab = len(s["score"]), s["width"], s["vocab"]
    z = s["logits"].float()
    if s["pen_rows"] is not None:
        p = s["pen_rows"][:, None]
        z = torch.where(_bits_of(s["bits"], vocab) > 0, torch.where(z < 0, z * p, z / p), z)
    if s["temp_rows"] is not None:
        z = z / s["temp_rows"][:, None]
    z = z.double()   # totals that nearly tie
    top = z.amax(dim=-1, keepdim=True)
    z = z - (torch.log(torch.exp(z - top).sum(dim=-1, keepdim=True)) + top)
    total = s["score"].double()[:, None] + z
    done = s["done"].bool()
    total[done] = -math.inf
    total[done, STOP] = s["score"].double()[done]
    total, at = torch.sort(total.view(-1, width * vocab), dim=-1, descending=True, stable=True)
    total, at = total[:, :width].reshape(-1), at[:, :width].reshape(-1)
    parent, token = at // vocab, at % vocab
    group = torch.arange(rows, device="cuda") // width * width
    source = group + parent
    was = s["done"][source]
    s["bits_out"].copy_(s["bits"][source])
    row = torch.arange(rows, device="cuda")
    add = torch.where((was > 0) | (token == STOP), 0, torch.bitwise_left_shift(torch.ones_like(token), token % 32))
    s["bits_out"][row, token // 32] |= torch.where(add >= 1 << 31, add - (1 << 32), add).int()
    return {"parent": parent.int(), "token": token.int(), "score": total.float(),
            "done": was | (token == STOP).to(torch.uint8), "bits": s["bits_out"], "tokens": s["tokens"][source]}


def _rows4(s, name):
    """(codes, scales) of the cache, [page, position, head, ...]: views, through which it may be written too."""
    x, e = s[name], s[name + "_scale"].permute(0, 3, 1, 2)
    return x.permute(0, 2, 1, 3) if name == "k" else x.permute(0, 3, 1, 2), e


def _unpacked(byte):
    return torch.stack([byte & 15, byte >> 4], dim=-1).flatten(-2)


def _plain_kv4(s):
    seq, pos = _positions(s, s["off"])
    page, at = s["table"].long()[seq, pos // s["page"]], pos % s["page"]
    seq, pos = _positions(s, s["back_off"])
    back, back_at = s["table"].long()[seq, pos // s["page"]], pos % s["page"]
    out = {}
    for name in ("k", "v"):
        code, e = _codes4(s[name + "_new"].float())
        codes, scales = _rows4(s, name)
        codes[page, at] = _nibbles(code)
        scales[page, at] = e
        out[name] = _values4(_unpacked(codes[back, back_at]), scales[back, back_at]).to(torch.bfloat16)
    return out


def _plain_attn4(s):
    """Every sequence padded to the longest one, scores and weights whole."""
    table, lens = s["table"].long().clamp_min(0), s["lens"].long()
    n_seqs, heads, dim, kv = len(lens), s["heads"], s["dim"], s["kv_heads"]
    off = torch.arange(n_seqs + 1, device="cuda") if s["off"] is None else s["off"].long()
    n, most = off[1:] - off[:-1], s["max_new"]
    k, v = (_values4(_unpacked(c[table]), e[table]).flatten(1, 2).transpose(1, 2)      # [seq, head, position, dim]
            for c, e in (_rows4(s, "k"), _rows4(s, "v")))
    row = torch.arange(most, device="cuda")
    real = row < n[:, None]
    q = s["q"].float()[(off[:-1, None] + row).clamp_max(len(s["q"]) - 1)]   # [seq, row, head, dim]
    q = q.transpose(1, 2).reshape(n_seqs, kv, heads // kv * most, dim)
    score = (q @ k.transpose(2, 3) * dim ** -0.5).view(n_seqs, kv, heads // kv, most, -1)
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= (lens - n)[:, None, None] + row[:, None]
    if s["first"] is not None:
        seen = seen & (key >= s["first"][:, None, None])
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))       # a row that sees nothing: zeros
    o = p.view(n_seqs, kv, heads // kv * most, -1) @ v
    return {"out": o.view(n_seqs, heads, most, dim).transpose(1, 2)[real].to(torch.bfloat16)}


# ---- one pass, the framework's -------------------------------------------------------

_context = None


def _package():
    at = os.path.abspath("mlx-confucius4-tts_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import c4s
    return c4s


def _ctx():
    """The program's library context (one per host thread)."""
    global _context
    if _context is None:
        _context = _package().Context(0)
    return _context


def _own(s):
    c, kind = _ctx(), s["kind"]
    if kind == "rope":
        c.rope(s["q"], s["k"], s["freq"], s["lens"], s["off"], q_out=s["q_out"], k_out=s["k_out"],
               pairs=s["layout"] == "pairs", scale=s["factor"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if kind == "pages":
        c.pages_trim(s["handle"], s["drop"])
        c.pages_grow(s["handle"], s["new"], s["off"], s["pos"], s["slot"])
        return {n: s[n] for n in ("table", "lens", "refs", "free", "off", "pos", "slot", "missing")}
    if kind == "fork":
        c.pages_trim(s["handle"], s["ones"])
        c.pages_fork(s["handle"], s["parent"], s["width"])
        c.pages_grow(s["handle"], copies=s["copies"])
        out = {n: s[n] for n in ("table", "lens", "refs", "free", "copies", "missing")}
        for i, (kv, t) in enumerate(zip(s["kv"], s["caches"])):
            c.kv_copy(kv, s["copies"])
            out.update({"%s%d" % (n, i): t[n] for n in ("k", "v", "k_scale", "v_scale") if t[n] is not None})
        return out
    if kind == "beam":
        c.beam_step(s["logits"], s["width"], s["score"], s["score_out"], s["parent"], s["token"], done=s["done"],
                    out_done=s["done_out"], stop_token=STOP, temp=s["temp_rows"], pen=s["pen_rows"],
                    hist_bits=s["bits"], out_hist_bits=s["bits_out"], states=[(s["tokens"], s["tokens_out"])])
        return {"parent": s["parent"], "token": s["token"], "score": s["score_out"], "done": s["done_out"],
                "bits": s["bits_out"], "tokens": s["tokens_out"]}
    if kind == "kv4":
        c.kv_append(s["cache"], s["k_new"], s["v_new"], s["lens"], s["off"])
        c.kv_read(s["cache"], s["k_out"], s["v_out"], s["lens"], s["back_off"])
        return {"k": s["k_out"], "v": s["v_out"]}
    c.attn(s["q"], s["cache"], s["lens"], s["out"], rows_off=s["off"], max_new=s["max_new"], first=s["first"])
    return {"out": s["out"]}


def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "pages": _plain_pages, "fork": _plain_fork, "beam": _plain_beam, "kv4": _plain_kv4,
            "attn4": _plain_attn4}[s["kind"]](s)


# ---- what a pass cannot do without --------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rope":
        new, _ = _lengths(case)
        heads = sum(new) * (case["heads"] + case["kv_heads"])
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": float(heads * case["dim"] * 2 * size), "flops": float(heads * case["rot"] * 3)}
    if kind == "pages":
        had, drop, new = _moves(case)
        page = case["page"]
        turned = sum(-(-h // page) - -(-(h - d) // page) for h, d in zip(had, drop))
        # table entry and count out and in; lengths, offsets, drops; a position and a slot a row; the free bits
        pool = sum(-(-h // page) for h in had) * case["spare"] / 8
        return {"bytes": float(turned * 16 + len(had) * 20 + sum(new) * 8 + pool), "flops": 0.0}
    if kind == "beam":
        rows, vocab = case["groups"] * case["width"], case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": float(rows * (vocab * size + 2 * -(-vocab // 32) * 4 + 8 * case["hist"])),
                "flops": float(rows * vocab * 4)}
    if kind == "fork":
        rows, page = case["groups"] * case["width"], case["page"]
        lens = _spread(case["past_lo"], case["past_hi"], case["groups"])
        table = sum(-(-n // page) for n in lens) * case["width"] * 8
        value = {"bf16": 2.0, "q8": 1.0 + 4.0 / case["dim"], "q4": 0.5 + 1.0 / 32}[case["store"]]
        # three of eight beams copy, the filled half of a page each, where a page is not just full
        moved = sum(n % page for n in lens) * case["width"] * 3 / 8 * case["layers"]
        return {"bytes": table + rows * 32.0 + moved * case["heads"] * case["dim"] * value * 4, "flops": 0.0}
    new, lens = _lengths(case)
    row = 2.0 * case["dim"] * (0.5 + 1.0 / 32)   # a position's keys and values in the cache, one head
    if kind == "kv4":
        heads, back = case["heads"], sum(new) if case["back"] == "new" else sum(lens)
        return {"bytes": heads * (sum(new) + back) * (4.0 * case["dim"] + row), "flops": 0.0}
    first = _firsts(case, lens)
    seen = sum(max(0, p + 1 - f) for n, t, f in zip(new, lens, first) for p in range(t - n, t))
    keys = sum(t - min(f, t) for t, f in zip(lens, first))
    return {"bytes": keys * case["kv_heads"] * row + 4.0 * sum(new) * case["heads"] * case["dim"],
            "flops": 4.0 * seen * case["heads"] * case["dim"]}


# ---- in 64 bits -----------------------------------------------------------------------

def _exact_rope(s, new, lens):
    pos = torch.cat([torch.arange(t - n, t) for n, t in zip(new, lens)]).double().cuda()
    turn = torch.polar(torch.full((1,), s["factor"], dtype=torch.float64, device="cuda"), torch.outer(pos, s["freq"]))
    out = {}
    for name in ("q", "k"):
        x = s[name].double().clone()
        part = x[..., :s["rot"]]
        if s["layout"] == "half":
            z = torch.complex(*part.chunk(2, dim=-1)) * turn[:, None]
            x[..., :s["rot"]] = torch.cat([z.real, z.imag], dim=-1)
        else:
            z = torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * turn[:, None]
            x[..., :s["rot"]] = torch.view_as_real(z).flatten(-2)
        out[name] = x
    return out


def _exact_beam(s):
    """Totals of the best; whole numbers are compared as they are."""
    z, width = s["logits"].double(), s["width"]
    if s["pen_rows"] is not None:
        seen = _bits_of(s["bits"], s["vocab"]).bool()
        z = torch.where(seen, z * torch.where(z < 0, s["pen"], 1.0 / s["pen"]), z)
    z = torch.log_softmax(z / s["temp"], dim=-1) + s["score"].double()[:, None]
    best = []
    for group in range(s["groups"]):
        rows = range(group * width, (group + 1) * width)
        found = [s["score"][r].double()[None] if s["done"][r] else z[r].topk(min(width, s["vocab"])).values for r in rows]
        best.append(torch.cat(found).sort(descending=True).values[:width])
    return {"parent": None, "token": None, "score": torch.cat(best), "done": None, "bits": None, "tokens": None}


def _exact_row4(x):
    """The nearest values that 4 bits can hold, by search over all of them."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    odd = torch.tensor([0.0, 1.0] * 4, dtype=torch.float64, device="cuda")
    block = x.double().reshape(-1, 32)
    scale = 2.0 ** torch.ceil(torch.log2(block.abs().amax(1, keepdim=True) / 6.0))
    a = (block / scale).abs()
    best, value = torch.full_like(a, math.inf), torch.zeros_like(a)
    for g, o in zip(grid, odd):
        far = (a - g).abs() + 1e-9 * o
        value = torch.where(far < best, g, value)
        best = torch.minimum(best, far)
    return (value * scale).copysign(block).reshape(x.shape)


def _exact_stored(s, name, seq, upto):
    """Positions 0 .. upto of one sequence as the cache stands for them: [head, position, dim]."""
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    grid = torch.tensor(grid + [-x for x in grid], dtype=torch.float64, device="cuda")
    pages = s["table"][seq, : -(-upto // s["page"])].long()
    byte = s[name][pages] if name == "k" else s[name][pages].transpose(2, 3)
    x = torch.empty((*byte.shape[:3], s["dim"]), dtype=torch.float64, device="cuda")
    x[..., 0::2], x[..., 1::2] = grid[(byte % 16).long()], grid[(byte // 16).long()]
    scale = 2.0 ** (s[name + "_scale"][pages].transpose(2, 3).double() - 127.0)
    return (x * scale.repeat_interleave(32, dim=3)).transpose(0, 1).flatten(1, 2)[:, :upto]


def _exact_kv4(s, new, lens):
    out = {"k": [], "v": []}
    for name in out:
        rows = _exact_row4(s[name + "_new"])
        at = 0
        for b, (n, t) in enumerate(zip(new, lens)):
            if s["back"] == "all" and t > n:
                out[name].append(_exact_stored(s, name, b, t - n).transpose(0, 1))
            out[name].append(rows[at:at + n])
            at += n
    return {name: torch.cat(x) for name, x in out.items()}


def _exact_attn4(s, case, new, lens):
    out, at, shared = [], 0, s["heads"] // s["kv_heads"]
    for b, (n, t, first) in enumerate(zip(new, lens, _firsts(case, lens))):
        k, v = (_exact_stored(s, name, b, t) for name in ("k", "v"))
        o = torch.zeros((n, s["heads"], s["dim"]), dtype=torch.float64, device="cuda")
        hidden = torch.arange(t, device="cuda") > torch.arange(t - n, t, device="cuda")[:, None]
        hidden |= torch.arange(t, device="cuda") < first
        empty = hidden.all(1)
        for h in range(s["heads"]):
            z = s["q"][at:at + n, h].double() @ k[h // shared].t() / math.sqrt(s["dim"])
            p = torch.softmax(z.masked_fill(hidden, -math.inf), dim=1)
            o[:, h] = p.masked_fill(empty[:, None], 0.0) @ v[h // shared]
        out.append(o)
        at += n
    return {"out": torch.cat(out)}


def exact(case, seed):
    kind = case["kind"]
    if kind in ("pages", "fork"):   # whole numbers, and values that are moved as they are
        return None
    s = prepare(case, seed)
    if kind == "beam":
        return _exact_beam(s)
    new, lens = _lengths(case)
    if kind == "rope":
        return _exact_rope(s, new, lens)
    return _exact_kv4(s, new, lens) if kind == "kv4" else _exact_attn4(s, case, new, lens)
