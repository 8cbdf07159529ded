"""The decoder layer's operators: what they are measured on.

Four kinds of call, together one layer of the decoder in front of the LM head:

* ``norm``   -- ``block_norm``: a block's output joins the residual stream (a norm behind the block, a gate, a
  scale), and the norm in front of the next block reads the result.
* ``linear`` -- ``linear``: product with bias, activation and residual; bf16 weights or 8-bit codes in groups.
* ``kv``     -- ``kv_append`` and ``kv_read``: new tokens' keys and values into the paged cache, as bf16 or as
  8-bit codes with a scale a token and head, and read back as the values that the cache stands for.
* ``attn``   -- ``attn``: the new tokens of every sequence over the paged cache, one a sequence or many.

A cache's pages hold ``page`` tokens of one head together: keys as [page][head][token][dim], values as
[page][head][dim][token]. Pages are handed out in no order, and what no token has written yet holds an earlier
sequence's values.
"""
import math
import os
import sys

import torch

own = False

LAYER, RMS = "layer", "rms"
EPS = 1e-5


def listed():
    return [
        # One utterance's AR step: the attention's output joins the stream, the norm in front of the MLP.
        {"name": "norm_1", "kind": "norm", "rows": 1, "dim": 1280, "stream": "f32", "norm": LAYER, "post": False,
         "gate": 0},
        # Prompts of a batch, a norm on both sides of the block and one gate a prompt.
        {"name": "norm_16400_gated", "kind": "norm", "rows": 16400, "dim": 1280, "stream": "bf16", "norm": RMS,
         "post": True, "gate": 205},
        # One utterance's AR step: queries, keys and values.
        {"name": "linear_1_qkv", "kind": "linear", "rows": 1, "inputs": 1280, "outputs": 3840, "weight": "bf16",
         "group": 0, "act": "none", "residual": False},
        # A batch's AR step, 8-bit weights, into the MLP.
        {"name": "linear_64_gelu_q8", "kind": "linear", "rows": 64, "inputs": 1280, "outputs": 5120, "weight": "q8",
         "group": 64, "act": "gelu", "residual": False},
        # The same step, out of the MLP onto the float32 stream: few columns, a long sum.
        {"name": "linear_64_residual", "kind": "linear", "rows": 64, "inputs": 5120, "outputs": 1280,
         "weight": "bf16", "group": 0, "act": "none", "residual": True},
        # The prompts of a batch, an odd number of tokens.
        {"name": "linear_12345_gelu", "kind": "linear", "rows": 12345, "inputs": 1280, "outputs": 5120,
         "weight": "bf16", "group": 0, "act": "gelu", "residual": False},
        # A batch's AR step: one token a row, quantised.
        {"name": "kv_64_q8", "kind": "kv", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 50, "past_hi": 900,
         "heads": 20, "dim": 64, "page": 16, "store": "q8", "back": "new"},
        # Prompts behind a prefix that the cache holds already; whole sequences go out to another worker.
        {"name": "kv_prompts_q8", "kind": "kv", "seqs": 24, "new_lo": 70, "new_hi": 1500, "past_lo": 0,
         "past_hi": 333, "heads": 20, "dim": 64, "page": 64, "store": "q8", "back": "all"},
        # One utterance's AR step near its start, where latency is everything.
        {"name": "attn_1", "kind": "attn", "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 200, "past_hi": 200,
         "heads": 20, "kv_heads": 20, "dim": 64, "page": 16, "store": "bf16", "left": False},
        # A batch's AR step, every row of its own length.
        {"name": "attn_64", "kind": "attn", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 50, "past_hi": 1500,
         "heads": 20, "kv_heads": 20, "dim": 64, "page": 16, "store": "bf16", "left": False},
        # Few long rows of a text model with shared heads, an 8-bit cache.
        {"name": "attn_6_long_q8", "kind": "attn", "seqs": 6, "new_lo": 1, "new_hi": 1, "past_lo": 12000,
         "past_hi": 50001, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "store": "q8", "left": False},
        # Prompts of a batch, some of them behind a prefix, some of them padded on the left.
        {"name": "attn_prompts", "kind": "attn", "seqs": 12, "new_lo": 500, "new_hi": 2100, "past_lo": 0,
         "past_hi": 300, "heads": 20, "kv_heads": 20, "dim": 64, "page": 16, "store": "bf16", "left": True},
    ]


def _log(rng, lo, hi, unit=1):
    """A multiple of `unit` from lo to hi (themselves multiples), uniform in its logarithm."""
    n = unit * int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / unit))
    return max(lo, min(hi, n if n != 3072 else n - unit))


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "kv", "attn", "attn"])
    if kind == "norm":
        # the stream's width, or any other, odd ones too
        dim = 1280 if rng.random() < 0.4 else _log(rng, 64, 8192)
        rows = min(_log(rng, 1, 16400), max(1, 16400 * 1280 // dim))
        return {"kind": kind, "rows": rows, "dim": dim, "stream": rng.choice(["f32", "bf16"]),
                "norm": rng.choice([LAYER, RMS]), "post": rng.random() < 0.5,
                "gate": rng.choice([0, _log(rng, 1, 512)])}
    if kind == "linear":
        weight = rng.choice(["bf16", "q8"])
        group = rng.choice([32, 64, 128]) if weight == "q8" else 0
        inputs = _log(rng, 256, 8192, 128 if weight == "q8" else 8)
        outputs = rng.choice([1280, 3840, 5120, _log(rng, 100, 8200)])
        rows = max(1, min(_log(rng, 1, 12345), 12345 * 1280 * 5120 // (inputs * outputs)))
        return {"kind": kind, "rows": rows, "inputs": inputs, "outputs": outputs, "weight": weight, "group": group,
                "act": rng.choice(["none", "gelu", "silu"]), "residual": rng.random() < 0.5}
    heads, kv_heads, dim = rng.choice([(20, 20, 64), (20, 20, 64), (16, 4, 128), (32, 8, 128), (16, 2, 64),
                                       (12, 12, 80), (10, 5, 256)])
    page, store = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "q8"])
    if kind == "kv":
        new = _log(rng, 1, 1500)
        past = _log(rng, 1, 1500)
        seqs = max(1, min(_log(rng, 1, 128), 24 * 950 * 20 * 64 // ((new + past) * kv_heads * dim)))
        return {"kind": kind, "seqs": seqs, "new_lo": max(1, new // 8), "new_hi": new, "past_lo": past // 8,
                "past_hi": past, "heads": kv_heads, "dim": dim, "page": page, "store": store,
                "back": rng.choice(["new", "all"])}
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "store": store,
         "left": rng.random() < 0.3}
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


def _quantised(x):
    """8-bit codes of rows of the last dimension, and their scales."""
    scale = x.abs().amax(dim=-1) / 127.0
    return torch.round(x / scale.clamp_min(1e-30)[..., None]).to(torch.int8), scale


def _cache(case, g, lens, heads):
    """The paged cache with every page written before: pages, scales, and each sequence's pages."""
    page, dim = case["page"], case["dim"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    c = {"table": table, "k_scale": None, "v_scale": None}
    for name in ("k", "v"):
        x = _randn(g, pages, heads, page, dim).to(torch.bfloat16)
        if case["store"] == "q8":
            x, scale = _quantised(x.float())
            c[name + "_scale"] = scale
        c[name] = x if name == "k" else x.transpose(2, 3).contiguous()
    return c


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = dict(case)
    if kind == "norm":
        rows, dim = case["rows"], case["dim"]
        t = torch.float32 if case["stream"] == "f32" else torch.bfloat16
        s["x"] = _randn(g, rows, dim).mul_(2.0).add_(0.3).to(t)
        s["y"] = _randn(g, rows, dim).to(torch.bfloat16)
        for name in ("gamma", "beta", "post_gamma", "post_beta"):
            s[name] = _randn(g, dim).mul_(0.05).add_(1.0 if "gamma" in name else 0.0)
        if case["norm"] == RMS:
            s["beta"] = s["post_beta"] = None
        if not case["post"]:
            s["post_gamma"] = s["post_beta"] = None
        s["g"] = _randn(g, -(-rows // case["gate"]), dim).mul_(0.3).add_(0.5) if case["gate"] else None
        s["scale"] = 0.75
        s["x_out"], s["out"] = torch.empty_like(s["x"]), torch.empty((rows, dim), dtype=torch.bfloat16, device="cuda")
    elif kind == "linear":
        rows, n, k = case["rows"], case["outputs"], case["inputs"]
        s["x"] = _randn(g, rows, k).to(torch.bfloat16)
        w = _randn(g, n, k).mul_(k ** -0.5)
        s["quant"] = None
        if case["weight"] == "q8":
            grp = w.view(n, k // case["group"], case["group"])
            lo, hi = grp.amin(dim=2), grp.amax(dim=2)
            scale = (hi - lo) / 255.0
            s["w"] = torch.round((grp - lo[..., None]) / scale[..., None]).clamp_(0, 255).to(torch.uint8).view(n, k)
            s["quant"] = (scale.contiguous(), lo.contiguous(), case["group"])
        else:
            s["w"] = w.to(torch.bfloat16)
        s["bias"] = _randn(g, n).mul_(0.1)
        s["res"] = _randn(g, rows, n) if case["residual"] else None
        s["out"] = torch.empty((rows, n), dtype=torch.float32 if case["residual"] else torch.bfloat16, device="cuda")
    else:
        new, lens = _lengths(case)
        total, heads, dim = sum(new), case.get("kv_heads", case["heads"]), case["dim"]
        s.update(_cache(case, g, lens, heads))
        s["lens"] = _ints(lens)
        one = max(new) == 1
        s["off"] = None if one else _ints([0] + torch.tensor(new).cumsum(0).tolist())
        s["max_new"] = max(new)
        if kind == "kv":
            # as a layer's product gives them: queries, keys and values side by side
            qkv = _randn(g, total, 3, heads, dim).to(torch.bfloat16)
            s["k_new"], s["v_new"] = qkv[:, 1], qkv[:, 2]
            s["back_off"] = s["off"] if case["back"] == "new" else _ints([0] + torch.tensor(lens).cumsum(0).tolist())
            n = total if case["back"] == "new" else sum(lens)
            s["k_out"], s["v_out"] = (torch.empty((n, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in "kv")
        else:
            s["q"] = _randn(g, total, case["heads"], dim).mul_(1.5).to(torch.bfloat16)
            s["first"] = _ints(_firsts(case, lens)) if case["left"] else None
            s["out"] = torch.empty_like(s["q"])
    if own and kind in ("kv", "attn"):   # the handle on the cache's tensors that a serving program holds
        s["cache"] = _package().KvCache(s["k"], s["v"], s["table"], s["k_scale"], s["v_scale"])
    return s


# ---- one pass, plain -----------------------------------------------------------------

def _norm(x, kind, gamma, beta):
    if kind == LAYER:
        x = x - x.mean(dim=-1, keepdim=True)
    x = x / (x.square().mean(dim=-1, keepdim=True) + EPS).sqrt() * gamma
    return x if beta is None else x + beta


def _plain_norm(s):
    u = s["y"].float()
    if s["post"]:
        u = _norm(u, s["norm"], s["post_gamma"], s["post_beta"])
    if s["gate"]:
        u = u * s["g"].repeat_interleave(s["gate"], dim=0)[:s["rows"]]
    r = s["x"].float() + s["scale"] * u
    return {"x": r.to(s["x"].dtype), "out": _norm(r, s["norm"], s["gamma"], s["beta"]).to(torch.bfloat16)}


def _act(y, act):
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y / (1.0 + torch.exp(-y)) if act == "silu" else y


def _plain_linear(s):
    w = s["w"].float()
    if s["quant"] is not None:
        scale, lo, group = s["quant"]
        w = (w.view(len(w), -1, group) * scale[..., None] + lo[..., None]).view(w.shape)
    y = _act(s["x"].float() @ w.t() + s["bias"], s["act"])
    if s["res"] is not None:
        y = y + s["res"]
    return {"out": y.to(s["out"].dtype)}


def _positions(s, off):
    """Of every row of the packed tensors with these offsets: its sequence, page and place in the page."""
    lens = s["lens"].long()
    off = torch.arange(len(lens) + 1, device="cuda") if off is None else off.long()
    n = off[1:] - off[:-1]
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), n)
    pos = lens[seq] - n[seq] + torch.arange(len(seq), device="cuda") - off[seq]
    return s["table"].long()[seq, pos // s["page"]], pos % s["page"]


def _plain_kv(s):
    page, at = _positions(s, s["off"])
    back = _positions(s, s["back_off"])
    out = {}
    for name in ("k", "v"):
        x = s[name + "_new"]
        if s["store"] == "q8":
            x, scale = _quantised(x.float())
            s[name + "_scale"][page, :, at] = scale
        cache = s[name] if name == "k" else s[name].transpose(2, 3)
        cache[page, :, at] = x
        y = cache[back[0], :, back[1]].float()
        if s["store"] == "q8":
            y = y * s[name + "_scale"][back[0], :, back[1]][..., None]
        out[name] = y.to(torch.bfloat16)
    return out


def _plain_attn(s):
    """Every sequence padded to the longest one, scores and weights whole."""
    table, lens = s["table"].long(), s["lens"].long()
    n_seqs, heads, dim, shared = len(lens), s["heads"], s["dim"], s["heads"] // s["kv_heads"]
    off = torch.arange(n_seqs + 1, device="cuda") if s["off"] is None else s["off"].long()
    n = off[1:] - off[:-1]
    k = s["k"][table].float()                       # [seq, page, head, token, dim]
    v = s["v"][table].float()                       # [seq, page, head, dim, token]
    if s["store"] == "q8":
        k = k * s["k_scale"][table][..., None]
        v = v * s["v_scale"][table][..., None, :]
    k = k.permute(0, 2, 1, 3, 4).reshape(n_seqs, s["kv_heads"], -1, dim)
    v = v.permute(0, 2, 1, 4, 3).reshape(n_seqs, s["kv_heads"], -1, dim)
    row = torch.arange(s["max_new"], device="cuda")
    real = row < n[:, None]
    q = s["q"].float()[(off[:-1, None] + row).clamp_max(len(s["q"]) - 1)]   # [seq, row, head, dim]
    q = q.view(n_seqs, s["max_new"], s["kv_heads"], shared, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(n_seqs, s["kv_heads"], shared * s["max_new"], dim)
    score = (q @ k.transpose(2, 3) * dim ** -0.5).view(n_seqs, s["kv_heads"], shared, s["max_new"], -1)
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= (lens - n)[:, None, None] + row[:, None]                   # [seq, row, key]
    if s["first"] is not None:
        seen = seen & (key >= s["first"][:, None, None])
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))       # a row that sees nothing: zeros
    o = p.view(n_seqs, s["kv_heads"], shared * s["max_new"], -1) @ v
    o = o.view(n_seqs, heads, s["max_new"], dim).transpose(1, 2)
    return {"out": o[real].to(torch.bfloat16)}


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
    if kind == "norm":
        c.block_norm(s["x"], s["gamma"], s["beta"], s["out"], y=s["y"], x_out=s["x_out"], post=s["post"],
                     post_gamma=s["post_gamma"], post_beta=s["post_beta"], gate=s["g"], gate_rows=s["gate"] or 1,
                     scale=s["scale"], eps=EPS, rms=s["norm"] == RMS)
        return {"x": s["x_out"], "out": s["out"]}
    if kind == "linear":
        c.linear(s["x"], s["w"], s["out"], bias=s["bias"], residual=s["res"], act=s["act"], quant=s["quant"])
        return {"out": s["out"]}
    if kind == "kv":
        c.kv_append(s["cache"], s["k_new"], s["v_new"], s["lens"], s["off"])
        c.kv_read(s["cache"], s["k_out"], s["v_out"], s["lens"], s["back_off"])
        return {"k": s["k_out"], "v": s["v_out"]}
    c.attn(s["q"], s["cache"], s["lens"], s["out"], rows_off=s["off"], max_new=s["max_new"], first=s["first"])
    return {"out": s["out"]}


def run(s):
    if own:
        return _own(s)
    return {"norm": _plain_norm, "linear": _plain_linear, "kv": _plain_kv, "attn": _plain_attn}[s["kind"]](s)


# ---- what a pass cannot do without --------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "norm":
        rows, dim = case["rows"], case["dim"]
        x = 4 if case["stream"] == "f32" else 2
        vectors = (1 if case["norm"] == RMS else 2) * (2 if case["post"] else 1)
        gates = -(-rows // case["gate"]) if case["gate"] else 0
        return {"bytes": float(rows * dim * (2 * x + 4) + 4 * dim * (vectors + gates)),
                "flops": float(rows * dim * (20 if case["post"] else 12))}
    if kind == "linear":
        m, n, k = case["rows"], case["outputs"], case["inputs"]
        w = 2.0 if case["weight"] == "bf16" else 1.0 + 8.0 / case["group"]
        return {"bytes": w * n * k + 2 * m * k + 4 * n + m * n * (8 if case["residual"] else 2),
                "flops": 2.0 * m * n * k}
    new, lens = _lengths(case)
    size = lambda heads: 2.0 * heads * (2 * case["dim"] if case["store"] == "bf16" else case["dim"] + 4)  # noqa: E731
    if kind == "kv":
        heads, back = case["heads"], sum(new) if case["back"] == "new" else sum(lens)
        plain = 4.0 * heads * case["dim"]
        return {"bytes": sum(new) * (plain + size(heads)) + back * (plain + size(heads)), "flops": 0.0}
    first = _firsts(case, lens)
    seen = sum(max(0, p + 1 - f) for n, t, f in zip(new, lens, first) for p in range(t - n, t))
    keys = sum(t - min(f, t) for t, f in zip(lens, first))
    return {"bytes": keys * size(case["kv_heads"]) + 4.0 * sum(new) * case["heads"] * case["dim"],
            "flops": 4.0 * seen * case["heads"] * case["dim"]}


# ---- in 64 bits -----------------------------------------------------------------------

def _exact_norm(s):
    def norm(x, gamma, beta):
        mean = x.mean(1, keepdim=True) if s["norm"] == LAYER else 0.0
        inv = torch.rsqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS)
        return (x - mean) * inv * gamma.double() + (0.0 if beta is None else beta.double())

    y = s["y"].double()
    if s["post"]:
        y = norm(y, s["post_gamma"], s["post_beta"])
    if s["gate"]:
        y = y * s["g"].double()[torch.arange(s["rows"], device="cuda") // s["gate"]]
    r = s["x"].double() + s["scale"] * y
    return {"x": r, "out": norm(r, s["gamma"], s["beta"])}


def _exact_linear(s):
    w = s["w"].double()
    if s["quant"] is not None:
        scale, lo, group = s["quant"]
        w = w * scale.double().repeat_interleave(group, 1) + lo.double().repeat_interleave(group, 1)
    y = torch.addmm(s["bias"].double(), s["x"].double(), w.t())
    if s["act"] == "gelu":
        y = y / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))
    elif s["act"] == "silu":
        y = y * torch.sigmoid(y)
    return {"out": y if s["res"] is None else s["res"].double() + y}


def _exact_stored(s, name, seq, upto):
    """Positions 0 .. upto of one sequence as the cache stands for them: [head, position, dim]."""
    pages = s["table"][seq, : -(-upto // s["page"])].long()
    x = s[name][pages].double()
    x = x if name == "k" else x.transpose(2, 3)
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][pages].double()[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :upto]


def _exact_kv(s, new, lens):
    out = {"k": [], "v": []}
    for name in out:
        rows = s[name + "_new"].double()
        if s["store"] == "q8":
            scale = rows.abs().amax(-1, keepdim=True) / 127
            rows = torch.round(rows / scale) * scale
        at = 0
        for b, (n, t) in enumerate(zip(new, lens)):
            if s["back"] == "all" and t > n:
                out[name].append(_exact_stored(s, name, b, t - n).transpose(0, 1))
            out[name].append(rows[at:at + n])
            at += n
    return {name: torch.cat(x) for name, x in out.items()}


def _exact_attn(s, case, new, lens):
    out, at = [], 0
    for b, (n, t, first) in enumerate(zip(new, lens, _firsts(case, lens))):
        shared = s["heads"] // s["kv_heads"]
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
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        return _exact_norm(s)
    if kind == "linear":
        return _exact_linear(s)
    new, lens = _lengths(case)
    return _exact_kv(s, new, lens) if kind == "kv" else _exact_attn(s, case, new, lens)
