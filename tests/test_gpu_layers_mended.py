"""Calls of the decoder layer's operators that once gave something else than their contract (include/c4s_layers.h)."""
import pytest
import torch

import c4s
import layers_util as L

pytestmark = pytest.mark.gpu


def _attn_raw(ctx, cache, lens, q, out, lse, off, n_rows, max_new, scale=0.125):
    """c4s_attn with every field as given."""
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    heads, dim = q.shape[1:]
    desc = c4s._pack_attn(p(q), heads * dim, p(out), heads * dim, p(lse), p(lens), p(off), 0, n_rows, max_new, heads, scale)
    return c4s.lib().c4s_attn(ctx._h, cache.packed, desc, torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("max_new", [0, -1, 1, 9, 2 ** 31 - 1])
def test_attn_without_offsets_has_one_row_a_sequence(gpu_ctx, max_new):
    """max_new means nothing without rows_off: a descriptor that leaves it zero computes all its rows."""
    cache = L.Cache([70, 3, 200], 2, 64, 16, False, seed=1)
    kc, lens = cache.cuda(), torch.tensor(cache.lens, dtype=torch.int32).cuda()
    q = L.bf16((3, 4, 64), torch.Generator().manual_seed(2)).cuda()
    out, lse = torch.full_like(q, 7.0), torch.full((3, 4), 7.0, device="cuda")
    assert _attn_raw(gpu_ctx, kc, lens, q, out, lse, None, 3, max_new) == c4s.OK
    want, wlse = torch.empty_like(q), torch.empty_like(lse)
    gpu_ctx.attn(q, kc, lens, want, max_new=1, lse=wlse)
    assert torch.equal(out, want) and torch.equal(lse, wlse) and (out != 7).any()


def test_attn_with_offsets_and_a_generous_max_new(gpu_ctx):
    """max_new above the rows there are says no more than their number."""
    cache = L.Cache([70, 40], 2, 64, 16, False, seed=1)
    kc, lens = cache.cuda(), torch.tensor(cache.lens, dtype=torch.int32).cuda()
    off = torch.tensor([0, 2, 5], dtype=torch.int32).cuda()
    q = L.bf16((5, 4, 64), torch.Generator().manual_seed(2)).cuda()
    want, got = torch.empty_like(q), torch.full_like(q, 7.0)
    gpu_ctx.attn(q, kc, lens, want, rows_off=off, max_new=5)
    for max_new in (6, 64, 2 ** 31 - 1):
        assert _attn_raw(gpu_ctx, kc, lens, q, got, None, off, 5, max_new) == c4s.OK
        assert torch.equal(got, want)
    assert _attn_raw(gpu_ctx, kc, lens, q, got.fill_(7.0), None, off, 5, 0) == c4s.OK
    assert (got == 7).all()   # nothing is to be computed
    assert _attn_raw(gpu_ctx, kc, lens, q, got, None, off, 5, -1) == c4s.EINVAL


def test_decoder_counts_its_room(gpu_ctx):
    """A step past the pages and positions that begin() gave is refused on the host (its position would be an index
    past the table of positions, which ends the process), and so is an id that is no token."""
    import c4s_decode as D

    w = D.random_weights(1, 128, 2, 1, 99, 20, seed=1)
    d = D.Decoder(gpu_ctx, w, 2, 1, 8)
    tokens = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="room"):
        d.step(tokens)
    d.begin([[1, 2, 3], [4] * 18], 2)
    for _ in range(2):
        assert torch.isfinite(d.step(tokens)).all()
    with pytest.raises(ValueError, match="room"):
        d.step(tokens)
    assert d.lens.tolist() == [5, 20]
    for prompts, new in (([[1, 99]], 1), ([[-1, 3]], 1), ([], 1), ([[1]], -1)):
        with pytest.raises(ValueError):
            d.begin(prompts, new)
        with pytest.raises(ValueError, match="room"):   # what began before is over
            d.step(tokens)
    one = lambda v, t: torch.full((1,), v, dtype=t, device="cuda")  # noqa: E731
    par = (one(0.9, torch.float32), one(5, torch.int32), one(0.9, torch.float32), one(1.0, torch.float32))
    with pytest.raises(ValueError):
        d.generate([[1, 2]], 0, *par, one(1, torch.int64))
    for n in (1, 2, 3, 18):   # up to the last position
        out = d.generate([[1, 2]], n, *par, one(7, torch.int64))
        assert out.shape == (1, n) and ((out >= 0) & (out < 99)).all()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("new,length,at", [
    (1, 300, 70), (1, 300, 290), (1, 33, 32), (1, 300, 0),     # single tokens: inside, in the last block, alone in it
    (5, 300, 70), (5, 300, 297), (5, 300, 295), (16, 300, 290),  # seen by some of the rows only, or by all
    (100, 300, 250), (1500, 1600, 800)])                       # prompts in either kernel
def test_values_that_are_not_finite_at_a_weight_of_zero(gpu_ctx, new, length, at, q8):
    """A seen position whose weight underflows still has a value: one that is not finite makes the rows that see it
    inf or NaN (0 times such a value), the other rows stay as they are."""
    heads, dim, page = 20 if new > 1000 else 2, 64, 16
    caches = [L.Cache([length], heads, dim, page, q8, seed=9) for _ in range(2)]
    for cache, bad in zip(caches, (True, False)):
        pg, place = int(cache.table[0, at // page]), at % page
        for name in cache.t:   # scores of every other position 0, of this one -512
            if name.startswith("k"):
                cache.t[name] = torch.zeros_like(cache.t[name])
        cache.t["k"][pg, :, place] = -127 if q8 else -8
        if q8:
            cache.t["k_scale"][pg, :, place] = 8 / 127
            if bad:
                cache.t["v_scale"][pg, :, place] = float("nan")
        elif bad:
            cache.t["v"][pg, :, 5, place] = float("inf")
            cache.t["v"][pg, :, 40, place] = float("nan")
    lens, off = torch.tensor([length], dtype=torch.int32).cuda(), torch.tensor([0, new], dtype=torch.int32).cuda()
    q = torch.ones((new, heads, dim), dtype=torch.bfloat16, device="cuda")
    got, want = torch.empty_like(q), torch.empty_like(q)
    for cache, out in zip(caches, (got, want)):
        gpu_ctx.attn(q, cache.cuda(), lens, out, rows_off=off, max_new=new, scale=1.0)
    assert torch.isfinite(want).all()
    sees = torch.arange(length - new, length, device="cuda") >= at
    odd = torch.ones(dim, dtype=torch.bool, device="cuda") if q8 else torch.zeros(dim, dtype=torch.bool, device="cuda")
    odd[5] = odd[40] = True
    assert not torch.isfinite(got[sees][:, :, odd]).any()
    assert torch.equal(got[sees][:, :, ~odd], want[sees][:, :, ~odd])
    assert torch.equal(got[~sees], want[~sees])


@pytest.mark.parametrize("M,N,K,group", [
    # few rows by outputs just above what the few rows' kernel took before by its count of tiles, and at it
    (1, 40960, 64, 0), (1, 40961, 64, 0), (16, 41000, 136, 0), (17, 41000, 136, 0), (64, 41003, 64, 0),
    (1, 41000, 4096, 0), (16, 41000, 4104, 0),
    (1, 51200, 64, 32), (1, 51201, 64, 64), (64, 51300, 128, 128), (65, 51300, 64, 32), (33, 60001, 96, 32)])
def test_linear_of_few_rows_and_many_outputs(gpu_ctx, M, N, K, group):
    print(f"linear {M}x{N}x{K} group={group}", flush=True)
    g = torch.Generator().manual_seed(M + N)
    x = L.bf16((M, K), g)
    quant = None
    if group:
        w = torch.randint(0, 256, (N, K), generator=g, dtype=torch.uint8)
        quant = (torch.rand((N, K // group), generator=g) * 0.02, torch.randn((N, K // group), generator=g), group)
    else:
        w = L.bf16((N, K), g)
    bias = torch.randn(N, generator=g)
    res = torch.randn((M, N), generator=g)
    want, err = L.linear(x, w, quant, bias, "silu", res)
    out = torch.empty((M, N), device="cuda")
    gpu_ctx.linear(x.cuda(), w.cuda(), out, bias=bias.cuda(), residual=res.cuda(), act="silu",
                   quant=None if quant is None else (quant[0].cuda(), quant[1].cuda(), group))
    bad = ~((L.f64(out) - want).abs() <= err)
    assert not bad.any(), f"{int(bad.sum())} off, first at {bad.nonzero()[0].tolist()}"
