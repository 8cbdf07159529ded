"""The decoder layer's operators where there is enough work to fill the chip: prompts
in attention's many-rows kernel, the cache's tiles of 64 rows, sequences of tens of
thousands of positions, and workspaces in graphs and on several streams. Bounds as
in test_gpu_layers.py."""
import numpy as np
import pytest
import torch

import c4s
import layers_util as L
from test_gpu_layers import _check_attn, _close, _packed, _run_attn

pytestmark = pytest.mark.gpu


def _fills(new, heads, kv_heads, seqs, q8=False, dim=64):
    """Tiles of 16 (row, query head) pairs of a key head: more than 700, and more than one a sequence
    (8-bit heads of up to 128: 1500, three)."""
    tiles = -(-max(new) * (heads // kv_heads) // 16)
    if q8 and dim <= 128:
        return tiles > 3 and tiles * kv_heads * seqs > 1500
    return tiles > 1 and tiles * kv_heads * seqs > 700


# ---- attention over prompts ---------------------------------------------------------------

PROMPTS = [  # new, past, heads, kv_heads, dim, page, q8
    ([210, 1, 64, 0, 129], [0, 50, 17, 3, 64], 20, 20, 64, 16, False),
    ([210, 1, 64, 0, 129], [7, 150, 17, 3, 63], 24, 24, 64, 32, True),
    ([190, 257], [300, 0], 32, 8, 48, 64, False),
    ([100, 31, 97], [29, 0, 200], 60, 20, 80, 128, False),
    ([150, 65], [3, 300], 80, 20, 128, 64, True),
    ([210, 1, 64, 70, 129], [7, 150, 17, 3, 63], 24, 24, 80, 16, True),
    ([400, 65], [3, 300], 32, 32, 48, 256, True),
    ([150, 65], [3, 300], 40, 10, 128, 16, False),
    ([70, 140], [7, 120], 40, 40, 256, 16, True),
    ([70, 140], [7, 120], 40, 40, 256, 256, False),
    ([61, 17, 40], [64, 1000, 0], 64, 16, 192, 32, False),
    ([260, 3, 50], [5, 90, 0], 32, 2, 112, 64, True),
    ([700], [1], 20, 20, 16, 16, False),
]


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,q8", PROMPTS)
def test_prompts(gpu_ctx, new, past, heads, kv_heads, dim, page, q8):
    """Unused places of the pages hold NaN."""
    print(f"attn prompts new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page} q8={q8}", flush=True)
    assert _fills(new, heads, kv_heads, len(new), q8, dim)
    cache = L.Cache([n + p for n, p in zip(new, past)], kv_heads, dim, page, q8, seed=dim + page, junk=float("nan"))
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads)
    _check_attn(cache, q, out, lse, new, heads, prompts=True)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_first(gpu_ctx, dim, q8):
    """Padding in front, in the middle of a block, past whole blocks, past every key of some rows or of all:
    zeros and an lse of -inf there. What is masked is not finite."""
    new, past, first, heads = [130, 100, 70, 20], [5, 130, 90, 0], [10, 131, 165, 2 ** 31 - 1], 48 if q8 else 32
    print(f"attn prompts first={first} dim={dim} q8={q8}", flush=True)
    assert _fills(new, heads, heads, 4, q8, dim)
    cache = L.Cache([n + p for n, p in zip(new, past)], heads, dim, 32, q8, seed=5, junk=float("inf"))
    for b, f in enumerate(first):
        for p in range(min(f, cache.lens[b])):
            pg, at = int(cache.table[b, p // 32]), p % 32
            for name in "kv":
                if q8:
                    cache.t[name + "_scale"][pg, :, at] = float("nan")
                elif name == "k":
                    cache.t["k"][pg, :, at] = float("nan")
                else:
                    cache.t["v"][pg, :, :, at] = float("inf")
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, first=first)
    empty = torch.cat([torch.arange(p, p + n) < f for n, p, f in zip(new, past, first)])
    assert empty.any() and (out.cpu()[empty] == 0).all() and torch.isinf(lse.cpu()[empty]).all()
    _check_attn(cache, q, out, lse, new, heads, first=first, prompts=True)


@pytest.mark.parametrize("q8", [False, True])
def test_prompts_missing_pages(gpu_ctx, q8):
    """Pages that are not there, one or several blocks of them, and a sequence of none; one longer than its table."""
    new, heads = [200, 30, 150, 90], 32 if q8 else 16
    assert _fills(new, heads, heads, 4, q8)
    cache = L.Cache([300, 30, 150, 100], heads, 64, 16, q8, seed=8)
    cache.table[0, 3:11] = -1
    cache.table[0, 14] = cache.n_pages + 5
    cache.table[1] = -1
    cache.table[2, 0] = -7
    cache.lens[0] = 320            # the table has pages for 304
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads)
    assert (out[200:230] == 0).all()
    _check_attn(cache, q, out, lse, new, heads, prompts=True)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n,p", [(700, 3), (640, 200)])
def test_prompts_later_rows_do_not_reach_earlier_ones(gpu_ctx, n, p, q8):
    """Keys and values that are not finite in later positions, up to two in a block of them."""
    heads = 40 if q8 else 20
    assert _fills([n], heads, heads, 1, q8)
    make = lambda: L.Cache([n + p], heads, 64, 16, q8, seed=6)  # noqa: E731
    cache, clean = make(), make()
    for bad in (p + n // 2, p + n // 2 + 2, p + n // 2 + 200):
        pg, at = int(cache.table[0, bad // 16]), bad % 16
        if q8:
            cache.t["v_scale"][pg, 0, at] = float("nan")
        else:
            cache.t["v"][pg, 0, 7, at] = float("nan")
            cache.t["v"][pg, 1, 9, at] = float("-inf")
            cache.t["k"][pg, 1, at, 3] = float("inf")
    q, out, lse = _run_attn(gpu_ctx, cache, [n], heads)
    o, h = out.cpu().float(), n // 2
    assert torch.isfinite(o[:h]).all() and torch.isfinite(o[:, 2:]).all()
    if q8:
        assert torch.isnan(o[h:, 0]).all()
    else:
        assert torch.isnan(o[h:, 0, 7]).all() and torch.isfinite(o[:, 0, :7]).all() and torch.isfinite(o[:, 0, 8:]).all()
    w, _, mag, sq = L.attn(clean, q[:, :], [n], heads, 0.125)
    err = 1e-4 * mag + 6 * 2.0 ** -9 * sq
    _close(out[:h], w[:h], err[:h])
    _close(out[:, 2:], w[:, 2:], err[:, 2:])


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 40.0])
def test_prompts_scales(gpu_ctx, scale):
    """No scores at all, negative ones, sharp ones, and scores of thousands (one key takes all)."""
    new, heads = [160, 90, 230], 20
    assert _fills(new, heads, heads, 3)
    cache = L.Cache([n + 100 for n in new], heads, 64, 16, False, seed=9)
    spread = 1.5 if scale < 40 else 0.25
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, scale=scale, spread=spread)
    if scale < 40:
        _check_attn(cache, q, out, lse, new, heads, scale=scale, prompts=True)
        return
    # scores of up to 40 * 8 * 0.25 * 4 = 320: their float32 error is 64 * 2^-24 of the products' magnitudes, below
    # 64 * 2^-24 * 40 * sum |q k| (below 60) = 0.01, relative in a weight and absolute in lse
    want, wlse, mag, sq = L.attn(cache, q, new, heads, scale)
    _close(out, want, 0.02 * mag + 6 * 2.0 ** -9 * sq)
    assert ((L.f64(lse) - wlse).abs() <= 0.01).all()


def _sampled(cache, q, out, lse, first_row, n, b, heads, rows, single):
    """Rows `rows` of sequence b's n against attn_row."""
    scale = cache.dim ** -0.5
    for i in rows:
        r = first_row + i
        want, wlse, mag, sq = L.attn_row(cache, b, cache.lens[b] - n + i, q[r], scale)
        _close(out[r], want, 1e-4 * mag + (6 * 2.0 ** -9 * sq if single else 0))
        assert ((L.f64(lse[r]) - wlse).abs() <= 1e-4).all()


@pytest.mark.parametrize("q8", [False, True])
def test_prompts_behind_long_prefixes(gpu_ctx, q8):
    """Prefixes of more pages than a workgroup looks up at a time (16384 positions), begun with the prefix or in it."""
    new, kv_heads = [50, 3, 64], 34 if q8 else 16
    heads = 4 * kv_heads
    assert _fills(new, heads, kv_heads, 3, q8)
    cache = L.Cache([33000, 40, 16384 + 30], kv_heads, 64, 16, q8, seed=3)
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, one=False)
    _sampled(cache, q, out, lse, 0, 50, 0, heads, [0, 17, 49], True)
    _sampled(cache, q, out, lse, 53, 64, 2, heads, [0, 33, 34, 63], True)
    new, heads = [64, 64], 190 if q8 else 90
    assert _fills(new, heads, heads, 2, q8)
    cache = L.Cache([16384 + 60, 200], heads, 32, 16, q8, seed=4)
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, one=False)
    _sampled(cache, q, out, lse, 0, 64, 0, heads, [0, 3, 4, 5, 63], True)
    _sampled(cache, q, out, lse, 64, 64, 1, heads, [0, 63], True)
    first = [16384 + 2, 0]
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, one=False, first=first)
    for i in (0, 1, 2, 5, 6, 63):
        want, wlse, mag, sq = L.attn_row(cache, 0, 16384 + 60 - 64 + i, q[i], 32 ** -0.5, first[0])
        _close(out[i], want, 1e-4 * mag + 6 * 2.0 ** -9 * sq)
        assert torch.equal(torch.isinf(lse[i].cpu()), torch.isinf(wlse))


# ---- single tokens over long and many sequences ----------------------------------------------

@pytest.mark.parametrize("q8", [False, True])
def test_few_rows_of_many_sequences_one_long(gpu_ctx, q8):
    """130 sequences fill the chip; one of them is longer than a workgroup's table of pages."""
    lens = [20000] + [1 + 3 * b for b in range(129)]
    cache = L.Cache(lens, 8, 64, 16, q8, seed=12)
    q, out, lse = _run_attn(gpu_ctx, cache, [1] * 130, 16)
    for b in (0, 1, 2, 6, 64, 129):
        _sampled(cache, q, out, lse, b, 1, b, 16, [0], False)


@pytest.mark.parametrize("new", [[1], [3]])
def test_few_rows_over_300000_positions(gpu_ctx, new):
    """As many parts of a sequence as there can be."""
    cache = L.Cache([300001], 1, 16, 256, False, seed=13, spare=0)
    q, out, lse = _run_attn(gpu_ctx, cache, new, 2, one=False)
    _sampled(cache, q, out, lse, 0, new[0], 0, 2, range(new[0]), False)


# ---- the cache, 64 rows a tile ---------------------------------------------------------------

KV = [  # new, past, heads, dim, page, q8
    ([500, 1, 0, 403], [0, 50, 3, 17], 20, 64, 16, False),
    ([500, 1, 0, 403], [0, 50, 3, 17], 20, 64, 64, True),
    ([1] * 300 + [400], [b % 70 for b in range(300)] + [11], 30, 64, 16, True),
    ([514, 2, 2], [126, 254, 1], 32, 128, 256, True),
    ([514, 2, 2], [126, 254, 1], 32, 128, 32, False),
    ([450, 3], [5, 31], 40, 256, 32, True),
    ([450, 3], [5, 31], 40, 208, 128, False),
    ([3] * 200, [b % 5 for b in range(200)], 30, 16, 16, False),
]


@pytest.mark.parametrize("new,past,heads,dim,page,q8", KV)
def test_kv_tiles(gpu_ctx, new, past, heads, dim, page, q8):
    """Codes, scales and bf16 values bit for bit, nothing else changed; reads give the rounded products. A page is
    missing, the rows begin at row 2 of the packed tensors, and what lies outside of them stays."""
    print(f"kv new={len(new)} rows={sum(new)} heads={heads} dim={dim} page={page} q8={q8}", flush=True)
    total = sum(new)
    assert (total + 5) // 64 * heads >= 256
    lens = [n + p for n, p in zip(new, past)]
    cache = L.Cache(lens, heads, dim, page, q8, seed=sum(lens))
    cache.table[0, min(1, cache.table.shape[1] - 1)] = cache.n_pages
    kc = cache.cuda()
    qkv = torch.randn((total + 5, 3, heads, dim), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    d = qkv.cuda()
    off = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)) + 2
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    gpu_ctx.kv_append(kc, d[:, 1], d[:, 2], lens_d, off.cuda())
    want = {k: v.clone() for k, v in cache.t.items()}
    for b, n in enumerate(new):
        pos = torch.arange(past[b], past[b] + n)
        pg, at = cache.table[b, pos // page].long(), pos % page
        there = pg < cache.n_pages
        pg, at, rows = pg[there], at[there], (torch.arange(n) + int(off[b]))[there]
        for i, name in ((1, "k"), (2, "v")):
            x = qkv[rows, i]
            if q8:
                x, s = L.quantise(x)
                want[name + "_scale"][pg, :, at] = s
            if name == "k":
                want["k"][pg, :, at] = x
            else:
                want["v"][pg, :, :, at] = x
    cache.update_from(kc)
    for name, t in want.items():
        assert torch.equal(t, cache.t[name]), name
    for t in (torch.bfloat16, torch.float32):
        k, v = (torch.full((total + 5, 2, heads, dim), 7.0, dtype=t, device="cuda")[:, 1] for _ in "kv")
        gpu_ctx.kv_read(kc, k, v, lens_d, off.cuda())
        for name, x in (("k", k.cpu()), ("v", v.cpu())):
            assert (x[:2] == 7).all() and (x[total + 2:] == 7).all()
            for b, n in enumerate(new):
                y, there = cache.rows(name, b, lens[b])
                y = torch.where(there[:, None, None], y, torch.zeros(())).to(torch.float32).to(t)[past[b]:]
                assert torch.equal(x[int(off[b]):int(off[b]) + n], y), (name, b)


@pytest.mark.parametrize("exponent", [-133, -126, -80, 0, 70, 119])
def test_kv_codes_of_every_mantissa(gpu_ctx, exponent):
    """Every pair of a row's largest magnitude and a value up to 2^-8 of it, as mantissas go: the codes of the
    definition's division, also where scales are subnormal or near the largest number."""
    top = torch.arange(128, 256).double() * 2.0 ** exponent                  # 128 mantissas of the largest magnitude
    val = torch.cat([torch.arange(128, 256).double() * 2.0 ** (exponent - e) for e in range(9)])
    rows = []
    for part in val.split(63):
        part = torch.cat([part, part.new_zeros(63 - len(part))])
        sign = torch.where(torch.arange(63) % 2 == 0, 1.0, -1.0)
        x = torch.minimum(part[None].expand(128, 63), top[:, None]) * sign
        rows.append(torch.cat([top[:, None], x], 1))
    x = torch.cat(rows).to(torch.bfloat16)[:, None]                          # [row][1 head][64]
    n = x.shape[0]
    cache = L.Cache([n], 1, 64, 64, True, seed=1)
    kc = cache.cuda()
    gpu_ctx.kv_append(kc, x.cuda(), (-x).cuda(), torch.tensor([n], dtype=torch.int32).cuda(),
                      torch.tensor([0, n], dtype=torch.int32).cuda())
    cache.update_from(kc)
    pos = torch.arange(n)
    pg, at = cache.table[0, pos // 64].long(), pos % 64
    q, s = L.quantise(x)
    assert torch.equal(cache.t["k_scale"][pg, :, at], s) and torch.equal(cache.t["v_scale"][pg, :, at], s)
    assert torch.equal(cache.t["k"][pg, :, at], q)
    assert torch.equal(cache.t["v"][pg, :, :, at], -q)


# ---- workspaces -------------------------------------------------------------------------------

def _split_state(seed, past=5000):
    """Inputs of a product split over K and of attention split over the length, both joined in a workspace."""
    g = torch.Generator().manual_seed(seed)
    bf = lambda *s: L.bf16(s, g, 0.1).cuda()  # noqa: E731
    lens = [past + 1, past // 3 + 1]
    cache = L.Cache(lens, 4, 64, 64, False, seed=seed)
    return dict(kc=cache.cuda(), lens=torch.tensor(lens, dtype=torch.int32).cuda(), q=bf(2, 4, 64), a=bf(2, 4, 64),
                x=bf(3, 5120), w=bf(1280, 5120), o=torch.empty((3, 1280), device="cuda"))


def _split(ctx, s):
    ctx.attn(s["q"], s["kc"], s["lens"], s["a"])
    ctx.linear(s["x"], s["w"], s["o"], act="gelu")
    return s["a"], s["o"]


def test_split_calls_in_a_graph_beside_eager_ones():
    """Replays with eager calls of other inputs and other streams between them: the same bits each time."""
    ctx = c4s.Context(0)
    s, other, third = _split_state(1), _split_state(2), _split_state(3, past=9000)
    want = [t.clone() for t in _split(ctx, s)]
    want2, want3 = ([t.clone() for t in _split(ctx, o)] for o in (other, third))
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _split(ctx, s)
        _split(ctx, s)
    more = [torch.cuda.Stream() for _ in range(3)]
    for st in more:
        st.wait_stream(torch.cuda.current_stream())
    for i in range(5):
        for t in (s["a"], s["o"]):
            t.zero_()
        graph.replay()
        _split(ctx, other)
        with torch.cuda.stream(more[i % 3]):
            _split(ctx, third)
        torch.cuda.synchronize()
        for o, w in ((s, want), (other, want2), (third, want3)):
            assert torch.equal(o["a"], w[0]) and torch.equal(o["o"], w[1]), i
    del graph
    torch.cuda.synchronize()
    ctx.close()


def test_a_workspace_does_not_grow_in_a_capture():
    """The first call of a size is refused there, and nothing of it is in the graph; made outside, it is captured."""
    ctx = c4s.Context(0)
    s = _split_state(4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        s["o"].zero_()
        with pytest.raises(c4s.C4SError, match="would grow"):
            ctx.linear(s["x"], s["w"], s["o"])
        with pytest.raises(c4s.C4SError, match="would grow"):
            ctx.attn(s["q"], s["kc"], s["lens"], s["a"])
    g.replay()
    torch.cuda.synchronize()
    assert (s["o"] == 0).all()
    want = [t.clone() for t in _split(ctx, s)]
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2, stream=side):
        _split(ctx, s)
    for _ in range(3):
        s["o"].zero_()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(s["a"], want[0]) and torch.equal(s["o"], want[1])
    del g, g2
    ctx.close()


def test_split_calls_on_two_streams_at_once(gpu_ctx):
    """Each stream joins in a workspace of its own."""
    a, b = _split_state(5), _split_state(6, past=12000)
    wa, wb = ([t.clone() for t in _split(gpu_ctx, s)] for s in (a, b))
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for st in (one, two):
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(30):
        for st, s in ((one, a), (two, b)):
            with torch.cuda.stream(st):
                _split(gpu_ctx, s)
    torch.cuda.synchronize()
    for s, w in ((a, wa), (b, wb)):
        assert torch.equal(s["a"], w[0]) and torch.equal(s["o"], w[1])


# ---- sizes ----------------------------------------------------------------------------------------

def test_norm_of_many_short_rows(gpu_ctx):
    """More rows than a grid's first dimension holds workgroups for (2^20 of four rows)."""
    M, D = (1 << 22) + 5, 3
    x = torch.randn((M, D), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = torch.empty((M, D), device="cuda")
    gpu_ctx.block_norm(x.cuda(), None, None, out)
    want = L.norm(L.f64(x), False, 1e-5, None, None)
    # deviations of three values: the mean's three roundings, twice an ulp of its products and the root
    err = 16 * L.U * (want.abs() + (L.f64(x).abs().amax(1) / (L.f64(x).var(1, unbiased=False) + 1e-5).sqrt())[:, None])
    assert ((L.f64(out) - want).abs() <= err).all()


def test_sizes_past_the_grid_are_refused(gpu_ctx):
    """Nothing is queued: the addresses are of small tensors."""
    z = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    kc = c4s.KvCache(z(3, 2, 16, 64), z(3, 2, 64, 16), z(2, 3, t=torch.int32))
    p, lens, off = z(16, 2, 64).data_ptr(), z(2, t=torch.int32).data_ptr(), z(3, t=torch.int32).data_ptr()
    rows = c4s._pack_rows(p, p, 128, 128, lens, off, (1 << 28) + 1, c4s.BF16)
    for call in (c4s.lib().c4s_kv_append, c4s.lib().c4s_kv_read):
        assert call(gpu_ctx._h, kc.packed, rows, None) == c4s.EINVAL
        assert b"536870912" in c4s.lib().c4s_last_error(gpu_ctx._h)
    n = (1 << 28) + 1
    attn = c4s._pack_attn(p, 128, p, 128, 0, lens, off, 0, n, n, 2, 0.125)
    assert c4s.lib().c4s_attn(gpu_ctx._h, kc.packed, attn, None) == c4s.EINVAL
    assert b"536870912" in c4s.lib().c4s_last_error(gpu_ctx._h)
    torch.cuda.synchronize()
