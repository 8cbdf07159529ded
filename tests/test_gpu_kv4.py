"""The cache in 4 bits (C4S_KV_Q4): codes and scales exactly, what is read back exactly, attention over it against
float64, with the bounds of test_gpu_layers.py (the values are bf16's, so its pages are like bf16 pages)."""
import math

import pytest
import torch

import batch_util as B
import c4s
import layers_util as L
from test_gpu_layers import _check_attn, _close, _packed, _run_attn

pytestmark = pytest.mark.gpu
I32, BF = torch.int32, torch.bfloat16


def _rows_of(kc, name, pg, at):
    """(codes [n][heads][dim], bytes [n][heads][dim / 32]) of a device cache."""
    t, s = getattr(kc, name).cpu(), getattr(kc, name + "_scale").cpu()
    byte = t[pg, :, at] if name == "k" else t[pg, :, :, at]
    return torch.stack([byte & 15, byte >> 4], -1).flatten(-2), s[pg, :, :, at]


KV = [  # new, past, heads, dim, page
    ([1] * 5, [0, 15, 16, 700, 63], 20, 64, 16),
    ([1], [3], 1, 32, 16),
    ([5, 0, 130, 1], [0, 7, 100, 33], 3, 96, 16),
    ([70, 1, 64], [13, 255, 0], 5, 256, 256),
    ([300, 41], [3, 1], 8, 128, 64),
    ([33, 31], [31, 2], 2, 160, 32),
    ([900], [7], 24, 64, 128),         # tiles of 64 rows
]


@pytest.mark.parametrize("new,past,heads,dim,page", KV)
def test_append_and_read(gpu_ctx, new, past, heads, dim, page):
    print(f"kv4 new={new} past={past} heads={heads} dim={dim} page={page}", flush=True)
    lens = [n + p for n, p in zip(new, past)]
    cache = B.Cache4(lens, heads, dim, page, seed=dim)
    kc = cache.cuda()
    g = torch.Generator().manual_seed(page)
    rows = torch.randn((sum(new), 3, heads, dim), generator=g) * torch.exp(2 * torch.randn((heads, dim), generator=g))
    rows = rows.to(BF)
    off = _packed(new, max(new) == min(new) == 1)
    off = None if off is None else off.cuda()
    ld = torch.tensor(lens, dtype=I32).cuda()
    d = rows.cuda()
    before = {n: getattr(kc, n).clone() for n in ("k", "v", "k_scale", "v_scale")}
    gpu_ctx.kv_append(kc, d[:, 1], d[:, 2], ld, off)
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)])
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)])
    pg, at = cache.table[seq, pos // page].long(), pos % page
    for i, name in ((1, "k"), (2, "v")):
        code, e = B.quantise4(rows[:, i])
        got = _rows_of(kc, name, pg, at)
        assert torch.equal(got[1], e) and torch.equal(got[0], code)
    # every other place as it was
    for name in "kv":
        t, s = getattr(kc, name), getattr(kc, name + "_scale")
        view = (lambda x: x) if name == "k" else (lambda x: x.transpose(2, 3))
        view(t)[pg.cuda(), :, at.cuda()] = view(before[name])[pg.cuda(), :, at.cuda()]
        s.transpose(2, 3)[pg.cuda(), :, at.cuda()] = before[name + "_scale"].transpose(2, 3)[pg.cuda(), :, at.cuda()]
        assert torch.equal(t, before[name]) and torch.equal(s, before[name + "_scale"])
    gpu_ctx.kv_append(kc, d[:, 1], d[:, 2], ld, off)
    cache.update_from(kc)
    # whole sequences back, as bf16 and as float32
    all_off = _packed(lens, False).cuda()
    for t in (BF, torch.float32):
        k, v = (torch.full((sum(lens) + 3, heads, dim), 7.0, dtype=t, device="cuda") for _ in "kv")
        gpu_ctx.kv_read(kc, k, v, ld, all_off)
        for name, x in (("k", k), ("v", v)):
            want = torch.cat([cache.rows(name, b, n)[0] for b, n in enumerate(lens)])
            assert torch.equal(L.f64(x[:sum(lens)]), want) and (x[sum(lens):] == 7).all()


def test_extremes(gpu_ctx):
    """Every bf16 value in every kind of block: alone, beside the largest there is, beside zeros, subnormal, not finite."""
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(BF)
    fine = every[torch.isfinite(every)]
    blocks = [fine[: len(fine) // 32 * 32].view(-1, 32)]                                  # neighbours in size
    blocks += [torch.cat([fine[i::257][:31], torch.tensor([t], dtype=BF)])[None] for i in range(0, 257, 9)
               for t in (3.3895313892515355e38, -1.0, 9.183549615799121e-41, 0.0, 6.0, 6.03125)]   # any beside one
    odd = torch.ones((3, 32), dtype=BF)
    odd[0, 5], odd[1, 31], odd[2, 0] = math.nan, math.inf, -math.inf
    x = torch.cat(blocks + [torch.zeros((1, 32), dtype=BF), -torch.zeros((1, 32), dtype=BF), odd])
    x = torch.cat([x, x[: -len(x) % 4]]).view(-1, 2, 64).contiguous()    # heads of 64: two blocks each
    n = len(x)
    table = torch.arange(-(-n // 16), dtype=I32).view(1, -1).cuda()
    kc = c4s.KvCache.empty(table.shape[1], 2, 16, 64, table, store="q4")
    lens, off = torch.tensor([n], dtype=I32).cuda(), torch.tensor([0, n], dtype=I32).cuda()
    d = x.cuda()
    gpu_ctx.kv_append(kc, d, d, lens, off)
    code, e = B.quantise4(x)
    at = torch.arange(n)
    for name in "kv":
        got = _rows_of(kc, name, at // 16, at % 16)
        assert torch.equal(got[1], e)
        real = (e != 255).repeat_interleave(32, -1)
        assert torch.equal(got[0][real], code[real])
    want = B.values4(code, e)
    for t in (BF, torch.float32):
        k, v = (torch.empty((n, 2, 64), dtype=t, device="cuda") for _ in "kv")
        gpu_ctx.kv_read(kc, k, v, lens, off)
        for got in (k, v):
            assert torch.equal(L.f64(got).nan_to_num(1.5), want.nan_to_num(1.5))
    step = torch.pow(2.0, e.double() - 127).repeat_interleave(32, -1)
    real = torch.isfinite(want)
    assert (x.double().abs()[torch.isinf(want)] >= 3.5 * 2.0 ** 126).all()
    assert ((want - x.double()).abs() <= step)[real].all()     # half of the widest step, from 4 to 6


ATTN = [  # new, past, heads, kv_heads, dim, page
    ([1] * 5, [0, 1, 63, 64, 700], 4, 4, 64, 16),
    ([1, 1, 1], [300, 17, 40], 32, 8, 128, 64),
    ([1], [129], 1, 1, 32, 16),
    ([3, 1, 4], [7, 100, 62], 12, 2, 96, 32),
    ([1, 2], [500, 3], 10, 5, 256, 16),
    ([5, 1], [33, 260], 3, 3, 160, 128),
    ([1, 8], [90, 1000], 16, 2, 64, 256),
    ([2, 1], [300, 20], 7, 1, 224, 64),
    ([2, 1, 0, 2], [70, 300, 5, 0], 3, 3, 64, 16),
    ([4, 3, 1], [100, 9, 0], 5, 5, 128, 32),
    ([1, 1], [65, 2], 9, 3, 160, 16),
    ([3], [1000], 2, 2, 256, 128),
]


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page", ATTN)
def test_attn_few_rows(gpu_ctx, new, past, heads, kv_heads, dim, page):
    """Unused places hold blocks that are not finite."""
    print(f"attn4 new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page}", flush=True)
    cache = B.Cache4([n + p for n, p in zip(new, past)], kv_heads, dim, page, seed=dim + page, junk=True)
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, spread=0.7)
    _check_attn(cache, q, out, lse, new, heads)


@pytest.mark.parametrize("new,heads", [([1, 1], 3), ([2, 1], 3), ([1, 1], 12), ([5, 1], 6)])
def test_attn_scales(gpu_ctx, new, heads):
    """No scale, negative ones, and scores that differ by hundreds, so that every block has a new greatest one; values
    of very different sizes beside each other."""
    for scale, spread, rising in ((0.0, 0.7, False), (-0.25, 0.7, False), (0.125, 5.0, False), (0.125, 1.0, True), (-0.125, 1.0, True)):
        print(f"attn4 scales {new} {heads} {scale} {spread} {rising}", flush=True)
        cache = B.Cache4([900, 333], 3, 64, 16, seed=21, junk=True)
        if rising:     # the first block of a key grows with its position, and so does the score of a q with ones there
            for b, n in enumerate(cache.lens):
                for p in range(n):
                    code, e = B.quantise4(torch.full((3, 32), float(p + 1)).to(BF))
                    pg, at = int(cache.table[b, p // 16]), p % 16
                    cache.t["k"][pg, :, at, :16] = code[:, 0::2] | code[:, 1::2] << 4
                    cache.t["k_scale"][pg, :, 0, at] = e[:, 0]
        for pg in range(cache.n_pages):
            cache.t["v_scale"][pg, :, 1] = torch.where(cache.t["v_scale"][pg, :, 1] < 253, 40 + 20 * (pg % 11), cache.t["v_scale"][pg, :, 1]).to(torch.uint8)
        g = torch.Generator().manual_seed(22)
        q = (torch.randn((sum(new), heads, 64), generator=g) * spread).to(BF)
        if rising:
            q[..., :32] = 1.0
        out = torch.empty((sum(new), heads, 64), dtype=BF, device="cuda")
        off = _packed(new, True)
        gpu_ctx.attn(q.cuda(), cache.cuda(), torch.tensor(cache.lens, dtype=I32).cuda(), out, rows_off=None if off is None else off.cuda(),
                     max_new=max(new), scale=scale)
        want, _, mag, _ = L.attn(cache, q, new, heads, scale)
        # scores of up to 500 in float32: 64 products' sum, 8 roundings of 2^-24 at most in a tree, the scale's: 3e-4 of a weight
        _close(out, want, (6e-4 if rising else 1e-4 if spread < 1 else 3e-4) * mag)


PROMPTS = [  # new, past, heads, kv_heads, dim, page
    ([210, 1, 64, 0, 129], [0, 50, 17, 3, 64], 20, 20, 64, 16),
    ([210, 1, 64, 70, 129], [7, 150, 17, 3, 63], 24, 24, 32, 32),
    ([190, 257], [300, 0], 32, 8, 64, 64),
    ([150, 65], [3, 300], 80, 20, 128, 64),
    ([100, 31, 97], [29, 0, 200], 60, 20, 96, 128),
    ([70, 140], [7, 120], 40, 40, 256, 16),
    ([61, 17, 40], [64, 1000, 0], 64, 16, 192, 256),
    ([40, 3], [0, 50], 4, 4, 64, 16),
    ([210, 1, 64, 70, 129], [0, 150, 17, 3, 63], 24, 24, 64, 16),
    ([100, 31, 97, 5], [29, 0, 200, 300], 80, 20, 96, 128),
]


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page", PROMPTS)
def test_attn_prompts(gpu_ctx, new, past, heads, kv_heads, dim, page):
    print(f"attn4 prompts new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page}", flush=True)
    cache = B.Cache4([n + p for n, p in zip(new, past)], kv_heads, dim, page, seed=dim + page, junk=True)
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, spread=0.7)
    _check_attn(cache, q, out, lse, new, heads, prompts=True)


@pytest.mark.parametrize("heads", [2, 40])
@pytest.mark.parametrize("new,past,first", [([1] * 6, [0, 10, 63, 64, 200, 700], [5, 0, 60, 65, 150, 1]),
                                            ([20, 70, 1, 3], [5, 130, 90, 0], [10, 131, 2, 100]),
                                            ([200, 3], [100, 600], [170, 2 ** 31 - 1])])
def test_attn_first(gpu_ctx, new, past, first, heads):
    """Padding in front, some rows left with nothing: zeros, and an lse of -inf. What is masked is not finite."""
    print(f"attn4 first={first} heads={heads}", flush=True)
    cache = B.Cache4([n + p for n, p in zip(new, past)], heads, 64, 16, seed=5, junk=True)
    for b, f in enumerate(first):
        for p in range(min(f, cache.lens[b])):
            cache.spoil("k", b, p)
            cache.spoil("v", b, p)
    q, out, lse = _run_attn(gpu_ctx, cache, new, 2 * heads, first=first, spread=0.7)
    want = L.attn(cache, q, new, 2 * heads, 0.125, first)[1]
    assert torch.isinf(want).any() and (out.cpu()[torch.isinf(want)] == 0).all()
    _check_attn(cache, q, out, lse, new, 2 * heads, first=first, prompts=True)


@pytest.mark.parametrize("n,past,heads", [(4, 70, 2), (100, 3, 2), (40, 200, 2), (700, 3, 20), (3, 600, 2), (700, 3, 40)])
def test_attn_later_rows_do_not_reach_earlier_ones(gpu_ctx, n, past, heads):
    """Blocks that are not finite in later positions: a value's own dims, and all of a row whose key it is."""
    mk = lambda: B.Cache4([n + past], heads, 64, 16, seed=6)  # noqa: E731
    cache, clean = mk(), mk()
    bad = past + n // 2
    cache.spoil("v", 0, bad, 0, 1)
    cache.spoil("k", 0, bad, 1, 0)
    q, out, lse = _run_attn(gpu_ctx, cache, [n], heads, spread=0.7)
    o, h = out.cpu().float(), n // 2
    assert torch.isfinite(o[:h]).all()
    assert torch.isnan(o[h:, 0, 32:]).all() and torch.isfinite(o[h:, 0, :32]).all() and torch.isnan(o[h:, 1]).all()
    assert torch.isfinite(o[:, 2:]).all()
    w, _, mag, sq = L.attn(clean, q, [n], heads, 0.125)
    _close(out[:h], w[:h], (1e-4 * mag + 6 * 2.0 ** -9 * sq)[:h])


def test_attn_a_value_that_is_not_finite_at_no_weight(gpu_ctx):
    """Rows that see it are NaN in its dims also where its weight underflows."""
    for n in (1, 4, 300, 700):
        heads = 2 if n < 100 else 40
        cache = B.Cache4([n + 200], heads, 64, 16, seed=7)
        cache.spoil("v", 0, 3, 1, 0)
        q = torch.zeros((n, 1, heads, 64), dtype=BF, device="cuda")
        q[..., 0] = 200.0
        k = cache.rows("k", 0, 200 + n)[0][:, 1, 0]      # make position 3 the least of all
        code, e = B.quantise4(torch.cat([torch.tensor([-60.0]), torch.zeros(31)]).to(BF))
        pg, at = int(cache.table[0, 0]), 3
        cache.t["k"][pg, 1, at, :16] = code[0::2] | code[1::2] << 4
        cache.t["k_scale"][pg, 1, 0, at] = e[0]
        assert (k[:3] > -50).all()
        out = torch.empty((n, heads, 64), dtype=BF, device="cuda")
        off = None if n == 1 else torch.tensor([0, n], dtype=I32).cuda()
        gpu_ctx.attn(q[:, 0], cache.cuda(), torch.tensor(cache.lens, dtype=I32).cuda(), out, rows_off=off)
        assert torch.isnan(out[:, 1, :32]).all() and torch.isfinite(out[:, 1, 32:]).all() and torch.isfinite(out[:, 0]).all()


@pytest.mark.parametrize("heads,new", [(2, [1, 1, 20]), (20, [200, 30, 150]), (60, [200, 30, 150])])
def test_attn_missing_pages(gpu_ctx, heads, new):
    cache = B.Cache4([300, 30, 150], heads, 64, 16, seed=8, junk=True)
    cache.table[0, 3:7] = -1
    cache.table[0, 12] = cache.n_pages + 5
    cache.table[1] = -1
    cache.table[2, 0] = -7
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, spread=0.7)
    assert (out[new[0]:new[0] + new[1]] == 0).all()
    _check_attn(cache, q, out, lse, new, heads, prompts=True)


def test_attn_long(gpu_ctx):
    for new in ([1, 1, 1], [4, 1, 3]):
        cache = B.Cache4([9001, 40, 700], 1, 64, 64, seed=10)
        q, out, lse = _run_attn(gpu_ctx, cache, new, 2, one=False, spread=0.7)
        _check_attn(cache, q, out, lse, new, 2)


def test_offsets_past_32_bits(gpu_ctx):
    """Pages whose bytes lie past 2^32."""
    heads, dim, page, n_pages = 16, 256, 256, 8300     # 4.35e9 bytes each
    small = B.Cache4([270, 70], heads, dim, page, seed=11, spare=0)
    table = small.table.clone()
    shift = n_pages - small.n_pages
    table[table >= 0] += shift
    kc = c4s.KvCache.empty(n_pages, heads, page, dim, table.cuda(), store="q4")
    for name in small.t:
        getattr(kc, name)[shift:] = small.t[name].cuda()
    g = torch.Generator().manual_seed(0)
    q, kv = L.bf16((4, heads, dim), g, 0.7), L.bf16((4, 2, heads, dim), g)
    lens, off = torch.tensor([270, 70], dtype=I32).cuda(), torch.tensor([0, 3, 4], dtype=I32).cuda()
    gpu_ctx.kv_append(kc, kv.cuda()[:, 0], kv.cuda()[:, 1], lens, off)
    out = torch.empty((4, heads, dim), dtype=BF, device="cuda")
    gpu_ctx.attn(q.cuda(), kc, lens, out, rows_off=off, max_new=3)
    for name in small.t:
        small.t[name] = getattr(kc, name)[shift:].cpu()
    for name, x in (("k", kv[:, 0]), ("v", kv[:, 1])):
        for r, (b, pos) in enumerate([(0, 267), (0, 268), (0, 269), (1, 69)]):
            assert torch.equal(small.row(name, b, pos), B.values4(*B.quantise4(x[r])))
    _check_attn(small, q, out, None, [3, 1], heads)


@pytest.mark.parametrize("new", [1, 40])
def test_in_a_graph_and_on_a_stream(gpu_ctx, new):
    """Rope, append and attention on another stream, captured, and replayed with eager work between: the same bits."""
    def state(seed):
        cache = B.Cache4([130 + new, 700 + new, new], 4, 64, 16, seed=seed)
        g = torch.Generator().manual_seed(seed)
        off = None if new == 1 else (torch.arange(4, dtype=I32) * new).cuda()
        return dict(kc=cache.cuda(), lens=torch.tensor(cache.lens, dtype=I32).cuda(), off=off,
                    qkv=L.bf16((3 * new, 16, 64), g).cuda(), out=torch.empty((3 * new, 8, 64), dtype=BF, device="cuda"))

    freq = c4s.rope_freqs(64)

    def run(s, stream=None):
        x = s["qkv"].clone() if stream is None else s["turned"]
        gpu_ctx.rope(x[:, :8], x[:, 8:12], freq, s["lens"], s["off"], stream=stream)
        gpu_ctx.kv_append(s["kc"], x[:, 8:12], x[:, 12:], s["lens"], s["off"], stream=stream)
        gpu_ctx.attn(x[:, :8], s["kc"], s["lens"], s["out"], rows_off=s["off"], max_new=new, stream=stream)

    a, b = state(1), state(2)
    run(a)
    torch.cuda.synchronize()
    want = a["out"].clone()
    side = torch.cuda.Stream()
    a["out"].zero_()
    a["turned"] = a["qkv"].clone()
    torch.cuda.synchronize()
    run(a, side)
    side.synchronize()
    assert torch.equal(a["out"], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(a)
    for _ in range(4):
        a["out"].zero_()
        graph.replay()
        run(b)
        torch.cuda.synchronize()
        assert torch.equal(a["out"], want)


def test_refusals(gpu_ctx):
    z = lambda *s, t=torch.uint8: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    table, lens = z(2, 3, t=I32), z(2, t=I32)
    for bad in (lambda: c4s.KvCache(z(3, 2, 16, 32), z(3, 2, 32, 16), table), lambda: c4s.KvCache(z(3, 2, 16, 32), z(3, 2, 64, 16), table, z(3, 2, 2, 16), z(3, 2, 2, 16)),
                lambda: c4s.KvCache(z(3, 2, 16, 32), z(3, 2, 32, 16), table, z(3, 2, 16, 2), z(3, 2, 16, 2)),
                lambda: c4s.KvCache(z(3, 2, 16, 32), z(3, 2, 32, 16), table, z(3, 2, 2, 16, t=torch.float32), z(3, 2, 2, 16, t=torch.float32)),
                lambda: c4s.KvCache.empty(3, 2, 16, 48, table, store="q4"), lambda: c4s.KvCache.empty(3, 2, 16, 64, table, store="q2")):
        with pytest.raises(ValueError):
            bad()
    kc = c4s.KvCache(z(3, 2, 16, 24), z(3, 2, 24, 16), table, z(3, 2, 1, 16), z(3, 2, 1, 16))    # heads of 48
    x = z(2, 2, 48, t=BF)
    for call in (lambda: gpu_ctx.attn(x, kc, lens, x), lambda: gpu_ctx.kv_append(kc, x, x, lens), lambda: gpu_ctx.kv_read(kc, x, x, lens),
                 lambda: gpu_ctx.kv_copy(kc, z(1, 2, t=I32))):
        with pytest.raises(c4s.C4SError, match="code 1.*multiple of 32"):
            call()
    torch.cuda.synchronize()
