"""The decoder layer's operators on the GPU against float64 (tests/layers_util.py).

Bounds: float32 sums in any order (linear: from K and the sums of magnitudes;
norms and softmax: a few dozen roundings), plus half a unit of a bf16 result
(one unit where a sum's error crosses a rounding boundary)."""
import numpy as np
import pytest
import torch

import c4s
import layers_util as L

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _close(got, want, err, out_dtype=torch.bfloat16):
    got = L.f64(got)
    bound = err + (L.BF16 * want.abs() if out_dtype == torch.bfloat16 else 0)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"got {got[bad][0].item()} want {want[bad][0].item()} bound {bound[bad][0].item()}")


# ---- block_norm ---------------------------------------------------------------------

NORMS = [  # M, D, x, y, out, rms, post, gate_rows (0: none), shift
    (1, 1280, "f32", "bf16", "bf16", False, False, 0, 0.0),
    (64, 1280, "f32", "bf16", "bf16", False, False, 0, 4.0),
    (37, 1280, "bf16", "bf16", "bf16", True, True, 5, 0.0),
    (3, 1, "f32", None, "f32", True, False, 0, 1.0),
    (5, 7, "bf16", "f32", "f32", False, True, 1, 0.0),
    (9, 1001, "f32", "bf16", "f32", False, True, 4, 1.0),
    (2, 2052, "bf16", None, "bf16", False, False, 0, 0.0),
    (3, 4099, "bf16", "bf16", "bf16", True, False, 2, 0.0),
    (2, 8196, "f32", "f32", "f32", True, True, 2, 0.0),
    (2, 16384, "bf16", "bf16", "bf16", False, True, 0, 0.0),
    (600, 512, "bf16", "bf16", "bf16", False, False, 600, 0.0),
    (1200, 1280, "f32", "bf16", "bf16", False, True, 100, 0.0),
]


@pytest.mark.parametrize("pad", [0, 1, 4])
@pytest.mark.parametrize("M,D,xt,yt,ot,rms,post,gate,shift", NORMS)
def test_block_norm(gpu_ctx, M, D, xt, yt, ot, rms, post, gate, shift, pad):
    print(f"block_norm {M}x{D} {xt} {yt} {ot} rms={rms} post={post} gate={gate} pad={pad}", flush=True)
    g = torch.Generator().manual_seed(M + D)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x = (rnd(M, D + pad) + shift).to(DT[xt])[:, :D]
    y = None if yt is None else (rnd(M, D + pad) * 0.5 + shift).to(DT[yt])[:, :D]
    gamma, beta = 1 + 0.1 * rnd(D), (None if rms else 0.1 * rnd(D))
    pg, pb = (1 + 0.1 * rnd(D), 0.1 * rnd(D)) if post else (None, None)
    gt = rnd(-(-M // gate), D) if gate else None
    dev = lambda t: None if t is None else torch.empty(t.shape[0], D + pad, dtype=t.dtype, device="cuda")[:, :D].copy_(t)  # noqa: E731
    xd, yd = dev(x), dev(y)
    xo = torch.full((M, D + pad), 7.0, dtype=DT[xt], device="cuda")
    out = torch.full((M, D + pad), 7.0, dtype=DT[ot], device="cuda")
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    gpu_ctx.block_norm(xd, c(gamma), c(beta), out[:, :D], y=yd, x_out=xo[:, :D], post=post, post_gamma=c(pg),
                       post_beta=c(pb), gate=c(gt), gate_rows=gate or 1, scale=0.75, eps=1e-5, rms=rms)
    u, uerr = None, 0.0
    r = L.f64(x)
    if y is not None:
        u = L.f64(y)
        uerr = torch.zeros_like(u)
        if post:
            uerr = 64 * L.U * (1 + shift + L.norm(u, rms, 1e-5, pg, pb).abs())
            u = L.norm(u, rms, 1e-5, pg, pb)
        f = 0.75 * (L.f64(gt)[torch.arange(M) // gate] if gate else 1.0)
        uerr = uerr * (f.abs() if gate else f) + 4 * L.U * (u * f).abs()
        r = r + f * u
    rerr = uerr + L.U * r.abs()
    _close(xo[:, :D], r, rerr, DT[xt])
    want = L.norm(r, rms, 1e-5, gamma, beta)
    std = (r - (0 if rms else r.mean(-1, keepdim=True))).square().mean(-1, keepdim=True).add(1e-5).sqrt()
    size = r.abs().amax(-1, keepdim=True) + (rerr.amax(-1, keepdim=True) / L.U if torch.is_tensor(rerr) else 0)
    _close(out[:, :D], want, 64 * L.U * (want.abs() + 1.5 * (size / std + 1)), DT[ot])
    if pad:
        assert (xo[:, D:] == 7).all() and (out[:, D:] == 7).all()


def test_block_norm_in_place_and_single_outputs(gpu_ctx):
    g = torch.Generator().manual_seed(3)
    x, y = torch.randn((33, 640), generator=g).cuda(), L.bf16((33, 640), g).cuda()
    gamma = torch.ones(640, device="cuda")
    a, oa = torch.empty_like(x), torch.empty((33, 640), dtype=torch.bfloat16, device="cuda")
    gpu_ctx.block_norm(x, gamma, None, oa, y=y, x_out=a)
    b, ob = x.clone(), torch.empty_like(oa)
    gpu_ctx.block_norm(b, gamma, None, ob, y=y, x_out=b)
    only = torch.empty_like(oa)
    gpu_ctx.block_norm(x, gamma, None, only, y=y)
    stream = torch.empty_like(x)
    gpu_ctx.block_norm(x, gamma, None, None, y=y, x_out=stream)
    assert torch.equal(a, b) and torch.equal(oa, ob) and torch.equal(oa, only) and torch.equal(a, stream)


def test_block_norm_constant_and_huge_rows(gpu_ctx):
    """A row without variance gives beta; a row far from zero loses no digits of its deviations."""
    D = 1280
    x = torch.full((2, D), 1000.0)
    x[1] += torch.arange(D) % 2            # deviations of 0.5 on a mean of 1000.5
    gamma, beta = torch.ones(D).cuda(), torch.full((D,), 0.25).cuda()
    out = torch.empty((2, D), device="cuda")
    gpu_ctx.block_norm(x.cuda(), gamma, beta, out)
    assert (out[0] == 0.25).all()
    _close(out[1], L.norm(x[1].double(), False, 1e-5, None, beta), torch.full((D,), 1e-4, dtype=torch.float64), torch.float32)


# ---- linear -----------------------------------------------------------------------------

LINEARS = [  # M, N, K, weight, group, act, residual, out, bias
    (1, 3840, 1280, "bf16", 0, "none", None, "bf16", True),
    (1, 100, 8, "bf16", 0, "gelu", None, "f32", False),
    (64, 5120, 1280, "q8", 64, "gelu", None, "bf16", True),
    (64, 1280, 5120, "bf16", 0, "none", "f32", "f32", True),
    (7, 1279, 5120, "q8", 128, "none", "f32", "f32", True),
    (16, 130, 1000, "bf16", 0, "silu", "bf16", "bf16", True),
    (17, 1, 64, "bf16", 0, "relu", None, "f32", True),
    (33, 515, 96, "q8", 32, "silu", "bf16", "f32", True),
    (65, 64, 2080, "bf16", 0, "gelu", "f32", "bf16", False),
    (130, 1280, 1288, "bf16", 0, "none", "f32", "f32", True),
    (300, 777, 640, "q8", 64, "relu", None, "bf16", False),
    (257, 3840, 1280, "bf16", 0, "gelu", None, "bf16", True),
    (1025, 515, 1288, "bf16", 0, "silu", "f32", "f32", True),
    (513, 1280, 1280, "q8", 32, "none", "bf16", "f32", True),
    (1500, 2560, 256, "bf16", 0, "none", "f32", "bf16", True),
    # tiles of many rows: 128 and 256 wide, the last ones partial, inputs that end inside a stage
    (2050, 1283, 1288, "bf16", 0, "silu", "f32", "f32", True),
    (2049, 1300, 8, "bf16", 0, "none", None, "f32", False),
    (4100, 2053, 72, "bf16", 0, "gelu", "bf16", "f32", True),
    (4099, 2052, 200, "bf16", 0, "relu", "f32", "bf16", False),
    (2600, 1281, 96, "q8", 32, "silu", "f32", "f32", True),
    (1300, 2560, 256, "q8", 128, "none", None, "bf16", True),
    (1411, 2564, 192, "q8", 64, "none", "bf16", "f32", False),
]


def _linear_inputs(M, N, K, weight, group, seed):
    g = torch.Generator().manual_seed(seed)
    x = L.bf16((M, K), g)
    w = torch.randn((N, K), generator=g) * K ** -0.5
    if weight == "bf16":
        return g, x, w.to(torch.bfloat16), None
    grp = w.view(N, K // group, group)
    lo, hi = grp.amin(2), grp.amax(2)
    scale = (hi - lo) / 255
    q = torch.round((grp - lo[..., None]) / scale[..., None]).clamp(0, 255).to(torch.uint8).view(N, K)
    return g, x, q, (scale.contiguous(), lo.contiguous(), group)


@pytest.mark.parametrize("M,N,K,weight,group,act,res,ot,bias", LINEARS)
def test_linear(gpu_ctx, M, N, K, weight, group, act, res, ot, bias):
    print(f"linear {M}x{N}x{K} {weight}/{group} {act} res={res} out={ot}", flush=True)
    g, x, w, quant = _linear_inputs(M, N, K, weight, group, M + N + K)
    b = 0.1 * torch.randn(N, generator=g) if bias else None
    r = None if res is None else torch.randn((M, N), generator=g).to(DT[res])
    out = torch.full((M, N + 3), 7.0, dtype=DT[ot], device="cuda")
    xd = torch.zeros((M, K + 8), dtype=torch.bfloat16, device="cuda")[:, :K].copy_(x)   # rows of a wider tensor
    gpu_ctx.linear(xd, w.cuda(), out[:, :N], bias=None if b is None else b.cuda(),
                   residual=None if r is None else r.cuda(), act=act,
                   quant=None if quant is None else (quant[0].cuda(), quant[1].cuda(), group))
    want, err = L.linear(x, w, quant, b, act, r)
    _close(out[:, :N], want, err, DT[ot])
    assert (out[:, N:] == 7).all()


@pytest.mark.parametrize("M,N", [(3, 256), (200, 256), (2100, 1400), (4100, 2100)])
def test_linear_in_place_residual(gpu_ctx, M, N):
    g, x, w, _ = _linear_inputs(M, N, 512, "bf16", 0, 5)
    r = torch.randn((M, N), generator=g).cuda()
    out = torch.empty_like(r)
    gpu_ctx.linear(x.cuda(), w.cuda(), out, residual=r)
    gpu_ctx.linear(x.cuda(), w.cuda(), r, residual=r)
    assert torch.equal(out, r)


@pytest.mark.parametrize("M,N", [(5, 200), (300, 200), (2600, 1300), (4100, 2100)])
@pytest.mark.parametrize("weight,group", [("bf16", 0), ("q8", 64)])
def test_linear_rows_do_not_touch_each_other(gpu_ctx, M, N, weight, group):
    """A row of NaN, inf or huge values leaves the other rows as they are, bit for bit."""
    _, x, w, quant = _linear_inputs(M, N, 256, weight, group, 9)
    q = None if quant is None else (quant[0].cuda(), quant[1].cuda(), group)
    a, b = (torch.empty((M, N), device="cuda") for _ in "ab")
    gpu_ctx.linear(x.cuda(), w.cuda(), a, act="gelu", quant=q)
    x[2] = torch.tensor([np.nan, np.inf, -np.inf, 3e38] * 64).to(torch.bfloat16)
    gpu_ctx.linear(x.cuda(), w.cuda(), b, act="gelu", quant=q)
    keep = torch.arange(M, device="cuda") != 2
    assert torch.equal(a[keep], b[keep]) and not torch.isfinite(b[2]).any()


# ---- the cache ------------------------------------------------------------------------------

KV = [  # new, past, heads, dim, page, q8
    ([1], [0], 1, 16, 16, False),
    ([1] * 9, [0, 1, 15, 16, 17, 31, 200, 63, 64], 20, 64, 16, True),
    ([1] * 5, [5, 0, 127, 128, 40], 3, 80, 32, False),
    ([0, 33, 1, 0, 100], [7, 3, 0, 0, 28], 2, 128, 64, True),
    ([17, 250, 16], [15, 0, 32], 4, 64, 16, False),
    ([129, 2], [130, 254], 1, 256, 256, True),
    ([40, 41, 0], [3, 9, 0], 5, 48, 128, False),
]


def _packed(n_new, one):
    off = np.concatenate([[0], np.cumsum(n_new)]).astype(np.int32)
    return None if one and all(n == 1 for n in n_new) else torch.from_numpy(off)


@pytest.mark.parametrize("new,past,heads,dim,page,q8", KV)
def test_kv_append_and_read(gpu_ctx, new, past, heads, dim, page, q8):
    """Codes, scales and bf16 values bit for bit; nothing else in the cache changes; reads give the rounded product."""
    print(f"kv new={new} past={past} heads={heads} dim={dim} page={page} q8={q8}", flush=True)
    lens = [n + p for n, p in zip(new, past)]
    cache = L.Cache(lens, heads, dim, page, q8, seed=sum(lens))
    kc = cache.cuda()
    g = torch.Generator().manual_seed(1)
    total = sum(new)
    qkv = torch.randn((total, 3, heads, dim), generator=g)
    qkv[total // 2, 1, 0] = 0.0                                     # a row of zeros
    qkv[total - 1, 2, heads - 1] *= 1e-20
    qkv = qkv.to(torch.bfloat16)
    d = qkv.cuda()
    off, lens_d = _packed(new, True), torch.tensor(lens, dtype=torch.int32).cuda()
    off = None if off is None else off.cuda()
    gpu_ctx.kv_append(kc, d[:, 1], d[:, 2], lens_d, off)
    want = {k: v.clone() for k, v in cache.t.items()}
    r = 0
    for b, n in enumerate(new):
        for i in range(n):
            pos = past[b] + i
            pg, at = int(cache.table[b, pos // page]), pos % page
            for name, x in (("k", qkv[r, 1]), ("v", qkv[r, 2])):
                if q8:
                    x, s = L.quantise(x)
                    want[name + "_scale"][pg, :, at] = s
                if name == "k":
                    want["k"][pg, :, at] = x
                else:
                    want["v"][pg, :, :, at] = x
            r += 1
    cache.update_from(kc)
    for name, t in want.items():
        assert torch.equal(t, cache.t[name]), name
    every = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
    for t in (torch.bfloat16, torch.float32):
        k, v = (torch.full((sum(lens) + 1, 2, heads, dim), 7.0, dtype=t, device="cuda")[:, 1] for _ in "kv")
        gpu_ctx.kv_read(kc, k, v, lens_d, every)
        r = 0
        for b, n in enumerate(lens):
            for pos in range(n):
                for name, x in (("k", k), ("v", v)):
                    # float32 product of code and scale, then one rounding
                    y = cache.row(name, b, pos).to(torch.float32).to(t)
                    assert torch.equal(x[r].cpu(), y), (name, b, pos)
                r += 1
        assert (k[-1] == 7).all() and (v[-1] == 7).all()


def test_kv_missing_pages(gpu_ctx):
    """Entries of the table outside the pages, and positions behind the table: not written, read as zeros."""
    cache = L.Cache([40, 20], 2, 64, 16, False, seed=1)
    cache.table[0, 1] = -1
    cache.table[1, 0] = cache.n_pages
    kc = cache.cuda()
    before = {k: v.clone() for k, v in cache.t.items()}
    lens = torch.tensor([40, 2000], dtype=torch.int32).cuda()      # sequence 1's last rows lie behind its table
    off = torch.tensor([0, 20, 25], dtype=torch.int32).cuda()
    rows = torch.full((25, 2, 64), 3.0, dtype=torch.bfloat16).cuda()
    gpu_ctx.kv_append(kc, rows, rows, lens, off)
    cache.update_from(kc)
    for p in range(cache.n_pages):
        hit = {(int(cache.table[0, 2]), a) for a in range(8)}
        for at in range(16):
            for name in "kv":
                x, y = (t[name][p, :, at] if name == "k" else t[name][p, :, :, at] for t in (cache.t, before))
                assert (x == 3).all() if (p, at) in hit else torch.equal(x, y)
    k, v = (torch.full((25, 2, 64), 7.0, device="cuda") for _ in "kv")
    gpu_ctx.kv_read(kc, k, v, lens, off)
    want = torch.zeros(25)
    want[12:20] = 3.0                                              # positions 32 .. 39 of sequence 0
    for x in (k, v):
        assert torch.equal(x.cpu(), want[:, None, None].expand(25, 2, 64))


def test_kv_non_finite_rows(gpu_ctx):
    """A value that is not finite makes NaN of its row of codes, and of no other."""
    cache = L.Cache([3, 3], 2, 64, 16, True, seed=2)
    kc = cache.cuda()
    x = L.bf16((2, 2, 64), torch.Generator().manual_seed(4))
    x[0, 1, 5], x[1, 0, 63] = float("inf"), float("nan")
    lens = torch.tensor([3, 3], dtype=torch.int32).cuda()
    gpu_ctx.kv_append(kc, x.cuda(), x.cuda(), lens)
    k, v = (torch.empty((2, 2, 64), device="cuda") for _ in "kv")
    gpu_ctx.kv_read(kc, k, v, lens)
    for t in (k, v):
        assert torch.isnan(t[0, 1]).all() and torch.isnan(t[1, 0]).all()
        assert torch.isfinite(t[0, 0]).all() and torch.isfinite(t[1, 1]).all()


# ---- attention --------------------------------------------------------------------------------

ATTN = [  # new, past, heads, kv_heads, dim, page, q8
    ([1], [0], 1, 1, 16, 16, False),
    ([1], [200], 20, 20, 64, 16, False),
    ([1] * 12, [0, 1, 14, 15, 16, 62, 63, 64, 127, 255, 256, 1000], 4, 4, 64, 16, False),
    ([1] * 12, [0, 1, 14, 15, 16, 62, 63, 64, 127, 255, 256, 1000], 4, 2, 64, 32, True),
    ([1, 1, 1], [700, 5, 2300], 32, 8, 128, 64, True),
    ([1, 1, 1], [700, 5, 2300], 16, 1, 128, 64, False),
    ([1, 1], [333, 90], 40, 2, 80, 128, False),
    ([1, 1], [333, 90], 6, 3, 48, 16, True),
    ([1, 1, 1], [600, 40, 0], 10, 5, 256, 256, False),
    ([1, 1], [600, 41], 10, 5, 256, 32, True),
    ([0, 3, 8, 1, 0], [10, 100, 0, 70, 0], 4, 4, 64, 16, False),
    ([5, 7], [300, 58], 12, 3, 128, 32, True),
    ([2, 4], [1500, 2], 8, 8, 96, 16, False),
]
PROMPTS = [
    ([33, 1, 200, 0, 64], [0, 50, 17, 3, 64], 4, 4, 64, 16, False),
    ([130, 257], [0, 300], 8, 2, 128, 64, False),
    ([130, 65], [3, 300], 4, 2, 64, 32, True),
    ([100, 31], [29, 0], 3, 1, 80, 128, False),
    ([48, 140], [7, 20], 4, 4, 256, 16, True),
    ([150], [1], 2, 2, 256, 16, False),
    ([17, 500], [1, 64], 6, 6, 64, 64, False),
    ([90, 160], [1, 64], 4, 2, 128, 16, True),
]


def _run_attn(ctx, cache, new, heads, seed=0, first=None, scale=None, one=True, spread=1.5, lse=True):
    g = torch.Generator().manual_seed(seed)
    total, dim = sum(new), cache.dim
    wide = (torch.randn((total, 2, heads, dim), generator=g) * spread).to(torch.bfloat16)   # q beside something else
    out = torch.full((total, 2, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ls = torch.full((total, heads), 7.0, device="cuda") if lse else None
    off = _packed(new, one)
    ctx.attn(wide.cuda()[:, 0], cache.cuda(), torch.tensor(cache.lens, dtype=torch.int32).cuda(), out[:, 1],
             rows_off=None if off is None else off.cuda(), max_new=max(new), scale=scale,
             first=None if first is None else torch.tensor(first, dtype=torch.int32).cuda(), lse=ls)
    assert (out[:, 0] == 7).all()
    return wide[:, 0], out[:, 1], ls


def _check_attn(cache, q, out, lse, new, heads, first=None, scale=None, prompts=False):
    want, wlse, mag, sq = L.attn(cache, q, new, heads, cache.dim ** -0.5 if scale is None else scale, first)
    # a score's float32 error, relative in its weight, and the weights' bf16 pairs: below 1e-4 of sum w |v|.
    # Prompts may round each weight to bf16 once: independent roundings of at most 2^-9, six sigma.
    err = 1e-4 * mag + (6 * 2.0 ** -9 * sq if prompts else 0)
    _close(out, want, err)
    if lse is not None:
        got = L.f64(lse)
        assert torch.equal(torch.isinf(got), torch.isinf(wlse))
        fine = torch.isfinite(wlse)
        assert ((got - wlse)[fine].abs() <= 1e-4).all()


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,q8", ATTN)
def test_attn_few_rows(gpu_ctx, new, past, heads, kv_heads, dim, page, q8):
    print(f"attn new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page} q8={q8}", flush=True)
    cache = L.Cache([n + p for n, p in zip(new, past)], kv_heads, dim, page, q8, seed=dim + page, junk=float("nan"))
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads)
    _check_attn(cache, q, out, lse, new, heads)


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,q8", PROMPTS)
def test_attn_prompts(gpu_ctx, new, past, heads, kv_heads, dim, page, q8):
    print(f"attn prompts new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page} q8={q8}", flush=True)
    cache = L.Cache([n + p for n, p in zip(new, past)], kv_heads, dim, page, q8, seed=dim + page, junk=float("nan"))
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads)
    _check_attn(cache, q, out, lse, new, heads, prompts=True)


MASKS = [([1] * 6, [0, 10, 63, 64, 200, 700], [5, 0, 60, 65, 150, 1]), ([20, 70, 1, 3], [5, 130, 90, 0], [10, 131, 2, 100]),
         ([200, 3], [100, 600], [170, 2 ** 31 - 1])]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("new,past,first", MASKS)
def test_attn_first(gpu_ctx, new, past, first, q8):
    """Padding in front, some rows left with nothing: zeros, and an lse of -inf. What is masked may be NaN."""
    print(f"attn first={first} q8={q8}", flush=True)
    cache = L.Cache([n + p for n, p in zip(new, past)], 2, 64, 16, q8, seed=5, junk=float("inf"))
    for b, f in enumerate(first):
        for p in range(min(f, cache.lens[b])):
            pg, at = int(cache.table[b, p // 16]), p % 16
            for name in "kv":
                if q8:
                    cache.t[name + "_scale"][pg, :, at] = float("nan")
                elif name == "k":
                    cache.t["k"][pg, :, at] = float("nan")
                else:
                    cache.t["v"][pg, :, :, at] = float("inf")
    q, out, lse = _run_attn(gpu_ctx, cache, new, 4, first=first)
    want = L.attn(cache, q, new, 4, 0.125, first)[1]
    assert torch.isinf(want).any()
    assert (out.cpu()[torch.isinf(want)] == 0).all()
    _check_attn(cache, q, out, lse, new, 4, first=first, prompts=True)


@pytest.mark.parametrize("new,past", [([4], [70]), ([100], [3]), ([40], [200])])
def test_attn_later_rows_do_not_reach_earlier_ones(gpu_ctx, new, past):
    """Keys and values that are not finite in a later position of the same block of new tokens."""
    n, p = new[0], past[0]
    cache = L.Cache([n + p], 2, 64, 16, False, seed=6)
    bad = p + n // 2
    pg, at = int(cache.table[0, bad // 16]), bad % 16
    cache.t["v"][pg, 0, 7, at] = float("nan")
    cache.t["v"][pg, 1, 9, at] = float("-inf")
    cache.t["k"][pg, 1, at, 3] = float("inf")
    q, out, lse = _run_attn(gpu_ctx, cache, new, 4)
    o = out.cpu().float()
    assert torch.isfinite(o[: n // 2]).all()
    assert not torch.isfinite(o[n // 2:, :2, 7]).any() and torch.isfinite(o[n // 2:, :2, :7]).all()
    short = L.Cache([n + p], 2, 64, 16, False, seed=6)      # the same cache without them
    w, _, mag, sq = L.attn(short, q, new, 4, 0.125)
    _close(out[: n // 2], w[: n // 2], (1e-4 * mag + 6 * 2.0 ** -9 * sq)[: n // 2])


@pytest.mark.parametrize("q8", [False, True])
def test_attn_missing_pages(gpu_ctx, q8):
    """Pages that are not there are not seen; a sequence of none of them gives zeros."""
    new = [1, 1, 20]
    cache = L.Cache([300, 30, 150], 2, 64, 16, q8, seed=8)
    cache.table[0, 3:7] = -1
    cache.table[0, 12] = cache.n_pages + 5
    cache.table[1] = -1
    cache.table[2, 0] = -7
    q, out, lse = _run_attn(gpu_ctx, cache, new, 4)
    assert (out[1] == 0).all()
    _check_attn(cache, q, out, lse, new, 4, prompts=True)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
@pytest.mark.parametrize("new", [[1, 1], [30, 90]])
def test_attn_scales(gpu_ctx, scale, new):
    """No scores at all, negative ones, and sharp ones (a weight of nearly one)."""
    cache = L.Cache([n + 100 for n in new], 2, 64, 16, False, seed=9)
    q, out, lse = _run_attn(gpu_ctx, cache, new, 2, scale=scale)
    _check_attn(cache, q, out, lse, new, 2, scale=scale, prompts=True)


def test_attn_long(gpu_ctx):
    """A sequence of 9001 tokens beside short ones, split over its length: one row and four."""
    for new in ([1, 1, 1], [4, 1, 3]):
        cache = L.Cache([9001, 40, 700], 1, 64, 64, False, seed=10)
        q, out, lse = _run_attn(gpu_ctx, cache, new, 2, one=False)
        _check_attn(cache, q, out, lse, new, 2)


@pytest.mark.parametrize("q8", [False, True])
def test_attn_offsets_past_32_bits(gpu_ctx, q8):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements of the cache."""
    heads, dim, page, n_pages = 16, 128, 64, 17000      # 2.2e9 elements each
    small = L.Cache([130, 70], heads, dim, page, q8, seed=11, spare=0)
    table = small.table.clone()
    shift = n_pages - small.n_pages
    table[table >= 0] += shift
    kc = c4s.KvCache.empty(n_pages, heads, page, dim, table.cuda(), q8=q8)
    for name in small.t:
        getattr(kc, name)[shift:] = small.t[name].cuda()
    g = torch.Generator().manual_seed(0)
    new = [3, 1]
    q = L.bf16((4, heads, dim), g)
    kv = L.bf16((4, 2, heads, dim), g)
    lens = torch.tensor([130, 70], dtype=torch.int32).cuda()
    off = torch.tensor([0, 3, 4], dtype=torch.int32).cuda()
    gpu_ctx.kv_append(kc, kv.cuda()[:, 0], kv.cuda()[:, 1], lens, off)
    out = torch.empty((4, heads, dim), dtype=torch.bfloat16, device="cuda")
    gpu_ctx.attn(q.cuda(), kc, lens, out, rows_off=off, max_new=3)
    k, v = (torch.empty((4, heads, dim), device="cuda") for _ in "kv")
    gpu_ctx.kv_read(kc, k, v, lens, off)
    for name in small.t:
        small.t[name] = getattr(kc, name)[shift:].cpu()
    for r, (b, pos) in enumerate([(0, 127), (0, 128), (0, 129), (1, 69)]):
        assert torch.equal(L.f64(k[r]), small.row("k", b, pos).float().double())
        assert torch.equal(L.f64(v[r]), small.row("v", b, pos).float().double())
    _check_attn(small, q, out, None, new, heads)


# ---- all of them ------------------------------------------------------------------------------

def _layer_state(seqs=3, new=1, seed=0, heads=4, dim=64):
    g = torch.Generator().manual_seed(seed)
    D = heads * dim
    lens = [20 + 7 * b + new for b in range(seqs)]
    cache = L.Cache(lens, heads, dim, 16, False, seed=seed)
    rows = seqs * new
    off = None if new == 1 else (torch.arange(seqs + 1, dtype=torch.int32) * new).cuda()
    bf = lambda *s: L.bf16(s, g, 0.1).cuda()  # noqa: E731
    return dict(D=D, rows=rows, heads=heads, dim=dim, kc=cache.cuda(), lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                off=off, new=new, x=torch.randn((rows, D), generator=g).cuda(), y=bf(rows, D), wqkv=bf(3 * D, D),
                wo=bf(D, D), gamma=torch.ones(D).cuda(), h=bf(rows, D), qkv=bf(rows, 3 * D), a=bf(rows, heads, dim),
                out=torch.empty((rows, D), device="cuda"))


def _layer(ctx, s):
    ctx.block_norm(s["x"], s["gamma"], None, s["h"], y=s["y"])
    ctx.linear(s["h"], s["wqkv"], s["qkv"])
    qkv = s["qkv"].view(s["rows"], 3, s["heads"], s["dim"])
    ctx.kv_append(s["kc"], qkv[:, 1], qkv[:, 2], s["lens"], s["off"])
    ctx.attn(qkv[:, 0], s["kc"], s["lens"], s["a"], rows_off=s["off"], max_new=s["new"])
    ctx.linear(s["a"].view(s["rows"], -1), s["wo"], s["out"], residual=s["x"])


@pytest.mark.parametrize("new", [1, 40])
def test_layer_on_another_stream_and_in_a_graph(gpu_ctx, new):
    """A layer's calls on a stream of the caller's, captured, and replayed with eager work in between: the same bits."""
    s = _layer_state(new=new)
    _layer(gpu_ctx, s)
    torch.cuda.synchronize()
    want = s["out"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s["out"].zero_()
        _layer(gpu_ctx, s)
        got = s["out"].clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _layer(gpu_ctx, s)
    other = _layer_state(new=new, seed=1)
    for _ in range(4):
        s["out"].zero_()
        graph.replay()
        _layer(gpu_ctx, other)
        torch.cuda.synchronize()
        assert torch.equal(s["out"], want)


@pytest.mark.parametrize("new", [1, 40])
def test_layer_gives_the_same_bits_twice(gpu_ctx, new):
    a, b = _layer_state(new=new, seqs=5), _layer_state(new=new, seqs=5)
    _layer(gpu_ctx, a)
    _layer(gpu_ctx, b)
    assert torch.equal(a["out"], b["out"])


# ---- refusals ---------------------------------------------------------------------------------

def test_refusals(gpu_ctx):
    z = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    f = torch.float32
    with pytest.raises(c4s.C4SError, match="code 1.*multiple of 8"):
        gpu_ctx.linear(z(2, 12), z(4, 12), z(2, 4))
    with pytest.raises(c4s.C4SError, match="code 1.*group"):
        gpu_ctx.linear(z(2, 96), z(4, 96, t=torch.uint8), z(2, 4), quant=(z(4, 2, t=f), z(4, 2, t=f), 48))
    with pytest.raises(c4s.C4SError, match="code 1.*16 bytes"):
        gpu_ctx.linear(z(2, 68)[:, 4:], z(4, 64), z(2, 4))
    for bad in (lambda: gpu_ctx.linear(z(2, 64, t=f), z(4, 64), z(2, 4)),
                lambda: gpu_ctx.linear(z(2, 64), z(4, 64, t=f), z(2, 4)),
                lambda: gpu_ctx.linear(z(2, 64), z(4, 64), z(2, 5)),
                lambda: gpu_ctx.linear(z(2, 64), z(4, 64), z(2, 4), act="tanh"),
                lambda: gpu_ctx.linear(z(2, 64), z(4, 64, t=torch.uint8), z(2, 4)),
                lambda: gpu_ctx.linear(z(2, 64), z(4, 64), z(2, 4), bias=z(5, t=f)),
                lambda: gpu_ctx.block_norm(z(2, 8), z(7, t=f), None, z(2, 8)),
                lambda: gpu_ctx.block_norm(z(2, 8), None, None, z(2, 8), y=z(3, 8)),
                lambda: gpu_ctx.block_norm(z(2, 8, t=torch.float16), None, None, z(2, 8)),
                lambda: c4s.KvCache(z(3, 2, 16, 64), z(3, 2, 16, 64), z(1, 3, t=torch.int32)),
                lambda: c4s.KvCache(z(3, 2, 16, 64, t=torch.int8), z(3, 2, 64, 16, t=torch.int8), z(1, 3, t=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(c4s.C4SError, match="code 1.*16384"):
        gpu_ctx.block_norm(z(1, 16385), None, None, z(1, 16385))
    with pytest.raises(c4s.C4SError, match="code 1.*without y"):
        gpu_ctx.block_norm(z(1, 8), None, None, z(1, 8), post=True)
    with pytest.raises(c4s.C4SError, match="code 1.*both outputs"):
        gpu_ctx.block_norm(z(1, 8), None, None, None)
    table, lens = z(2, 3, t=torch.int32), z(2, t=torch.int32)
    for size, dim, what in ((24, 64, "page_size"), (8, 64, "page_size"), (512, 64, "page_size"), (16, 24, "head_dim"),
                            (16, 272, "head_dim")):
        kc = c4s.KvCache(z(3, 2, size, dim), z(3, 2, dim, size), table)
        with pytest.raises(c4s.C4SError, match=f"code 1.*{what}"):
            gpu_ctx.attn(z(2, 2, dim), kc, lens, z(2, 2, dim))
        with pytest.raises(c4s.C4SError, match=f"code 1.*{what}"):
            gpu_ctx.kv_append(kc, z(2, 2, dim), z(2, 2, dim), lens)
    kc = c4s.KvCache(z(3, 2, 16, 64), z(3, 2, 64, 16), table)
    with pytest.raises(c4s.C4SError, match="code 1.*multiple of n_kv_heads"):
        gpu_ctx.attn(z(2, 3, 64), kc, lens, z(2, 3, 64))
    with pytest.raises(c4s.C4SError, match="code 1.*more rows than sequences"):
        gpu_ctx.attn(z(3, 2, 64), kc, lens, z(3, 2, 64))
    with pytest.raises(c4s.C4SError, match="code 1.*scale"):
        gpu_ctx.attn(z(2, 2, 64), kc, lens, z(2, 2, 64), scale=float("nan"))
    with pytest.raises(c4s.C4SError, match="code 1.*rows are bf16"):
        gpu_ctx.kv_append(kc, z(2, 2, 64, t=f), z(2, 2, 64, t=f), lens)
    for bad in (lambda: gpu_ctx.attn(z(2, 2, 64), kc, z(3, t=torch.int32), z(2, 2, 64)),
                lambda: gpu_ctx.attn(z(2, 2, 64), kc, z(2, t=torch.int64), z(2, 2, 64)),
                lambda: gpu_ctx.attn(z(2, 2, 128), kc, lens, z(2, 2, 128)),
                lambda: gpu_ctx.kv_read(kc, z(2, 3, 64), z(2, 3, 64), lens)):
        with pytest.raises(ValueError):
            bad()
    torch.cuda.synchronize()


def test_no_rows(gpu_ctx):
    z = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    kc = c4s.KvCache(z(3, 2, 16, 64), z(3, 2, 64, 16), z(2, 3, t=torch.int32))
    lens, off = z(2, t=torch.int32), z(3, t=torch.int32)
    gpu_ctx.linear(z(0, 64), z(4, 64), z(0, 4))
    gpu_ctx.block_norm(z(0, 64), None, None, z(0, 64))
    gpu_ctx.kv_append(kc, z(0, 2, 64), z(0, 2, 64), lens, off)
    gpu_ctx.kv_read(kc, z(0, 2, 64), z(0, 2, 64), lens, off)
    gpu_ctx.attn(z(0, 2, 64), kc, lens, z(0, 2, 64), rows_off=off)
    torch.cuda.synchronize()
