"""Rotary positions, pages handed out on the device, 4-bit pages and beam search together, as the decoder runs them
(c4s_decode.py): hidden rows against the decoder in float64, and a search against one whose hypotheses share nothing."""
import math

import numpy as np
import pytest
import torch

import batch_util as B
import c4s
import c4s_decode as D
import layers_util as L

pytestmark = pytest.mark.gpu

VOCAB = 515


def _decoder(ctx, store, rope, heads=8, kv_heads=4, layers=3, n_pages=200, page=16):
    w = D.random_weights(layers, heads * 64, heads, kv_heads, VOCAB, 400, seed=7, rope=rope)
    for l in w["layers"]:   # blocks that weigh as much as the embeddings
        for k in ("qkv", "out", "up", "down"):
            l[k] = (l[k].float() * 3).bfloat16()
    w["head"] = (w["head"].float() * 3).bfloat16()
    return D.Decoder(ctx, w, heads, kv_heads, n_pages, page, store=store)


def _reference(w, ids, heads, kv_heads):
    """Residual rows of one sequence after the last layer, float64 on the CPU, positions rotary."""
    x = L.f64(w["tokens"][ids])
    n, hd = len(ids), x.shape[1] // heads
    ln = lambda v, p: L.norm(v, False, 1e-5, *p)  # noqa: E731
    turn = lambda v: B.rope(v, torch.arange(n), w["rope"], False, 1.0)[0]  # noqa: E731
    mask = torch.full((n, n), float("-inf"), dtype=torch.float64).triu(1)
    for l in w["layers"]:
        qkv = (ln(x, l["norm1"]) @ L.f64(l["qkv"]).t() + L.f64(l["qkv_bias"])).view(n, heads + 2 * kv_heads, hd)
        q, k, v = turn(qkv[:, :heads]), turn(qkv[:, heads:heads + kv_heads]), qkv[:, heads + kv_heads:]
        k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        s = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) * hd ** -0.5 + mask, -1)
        a = torch.einsum("hij,jhd->ihd", s, v).reshape(n, -1)
        x = x + a @ L.f64(l["out"]).t() + L.f64(l["out_bias"])
        m = L.gelu(ln(x, l["norm2"]) @ L.f64(l["up"]).t() + L.f64(l["up_bias"]))
        x = x + m @ L.f64(l["down"]).t() + L.f64(l["down_bias"])
    return x


# bf16 roundings of 2^-9 at most: six a block at most (norm, products, rotation, weights), six blocks and the result,
# independent: sqrt(37) 2^-9 = 1.2 % of the row's length if all of it went through every one. 4-bit keys and values: the
# scale is below a third of the greatest of 32 normal numbers, 2.6 deviations as a rule: 0.87; codes are half a scale apart up
# to two, then a whole one (and two from four scales on, which is 3.5 deviations): 92 % of the numbers are off by
# 0.87 / 2 / sqrt(12), 8 % by twice that: 14 % of a deviation, twice a layer, three layers: 34 %.
BOUND = {"bf16": 0.012, "q8": 0.026, "q4": 0.35}


@pytest.mark.parametrize("store", ["bf16", "q8", "q4"])
def test_rotary_prompts_and_steps_against_float64(gpu_ctx, store):
    d = _decoder(gpu_ctx, store, True)
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randint(0, VOCAB, (n,), generator=g) for n in (90, 17, 213)]
    want = [_reference(d.w, s, d.heads, d.kv_heads) for s in seqs]
    for cut in (0, 1, 6):   # the last `cut` tokens one by one
        h = d.begin([s[:len(s) - cut] for s in seqs], cut + 1)
        for i in range(cut, 0, -1):
            h = d.step(torch.stack([s[-i] for s in seqs]).cuda())
        for got, x in zip(h, want):
            err = (L.f64(got) - x[-1]).norm() / x[-1].norm()
            print(f"{store} cut={cut}: {err:.4f}", flush=True)
            assert err <= BOUND[store]


def _unshared(d, prompts, width, max_new, stop, pen, temp):
    """The same search with all pages a hypothesis's own, copied whole, and the beams found in float64 on the CPU. Its calls
    of the layers have the shapes of the decoder's own, so that their results are the same to the bit."""
    n, R, ctx, w = [len(p) for p in prompts], len(prompts) * width, d.ctx, d.w
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(R * (-(-(max(n) + max_new) // d.page_size)), **i32).view(R, -1)
    caches = [c4s.KvCache.empty(table.numel(), d.kv_heads, d.page_size, d.hd, table,
                                store={torch.bfloat16: "bf16", torch.int8: "q8", torch.uint8: "q4"}[c.k.dtype]) for c in d.caches]
    for c in caches:
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            if t is not None:
                t.zero_()
    d.caches = caches
    lens = torch.zeros(R, dtype=torch.int32)
    lens[::width] = torch.tensor(n, dtype=torch.int32)
    off = torch.zeros(R + 1, dtype=torch.int32)
    off[1:] = lens.cumsum(0)
    d.lens = lens.cuda()
    b = d._buffers(sum(n))
    d._embed(b, torch.cat([torch.as_tensor(p) for p in prompts]).cuda(), torch.cat([torch.arange(k) for k in n]).cuda())
    d._layers(b, off.cuda(), max(n))
    h = b["x"].bfloat16()[(off[1::width] - 1).cuda().long()].repeat_interleave(width, 0).contiguous()
    d.lens = torch.tensor(n, **i32).repeat_interleave(width)
    d.one, d.room = d._buffers(R), max_new
    score = np.where(np.arange(R) % width == 0, 0.0, -np.inf).astype(np.float32)
    done, bits = np.zeros(R, bool), np.zeros((R, VOCAB), bool)
    out = np.zeros((R, max_new), np.int64)
    logits = torch.empty((R, VOCAB), device="cuda")
    for i in range(max_new):
        ctx.lmhead(h, *w["final_norm"], w["head"], w["head_bias"], logits)
        parent, token, total, done, bits = B.beams(logits.cpu().numpy(), width, score, done if stop >= 0 else None, stop,
                                                   np.full(R, temp, np.float32), np.full(R, pen, np.float32), bits)
        src = np.arange(R) // width * width + parent
        out = out[src]
        out[:, i] = token
        score = total.astype(np.float32)
        src = torch.from_numpy(src).cuda() if i else torch.arange(R, device="cuda") // width * width
        for c in caches:
            for t in (c.k, c.v, c.k_scale, c.v_scale):
                if t is not None:
                    t[table.long()] = t[table.long()[src]]
        h = d.step(torch.from_numpy(token).cuda())
    return out, score


SEARCH = [  # prompts, width, max_new, store, rope, stop, penalty, temperature, page
    ((30, 1, 77, 5), 4, 30, "q4", True, -1, 1.0, 1.0, 16),
    ((30, 16, 77, 5), 3, 20, "q8", False, 7, 1.3, 0.8, 16),
    ((64, 63), 8, 70, "bf16", True, 7, 1.0, 1.0, 64),
    ((200,), 32, 12, "q4", True, 7, 1.2, 1.5, 32),
    ((15, 31, 33), 1, 20, "q4", False, -1, 1.0, 1.0, 16),
    ((9,), 2, 1, "q4", True, -1, 1.0, 1.0, 16),
]


@pytest.mark.parametrize("lens,width,new,store,rope,stop,pen,temp,page", SEARCH)
def test_search_against_one_that_shares_nothing(gpu_ctx, lens, width, new, store, rope, stop, pen, temp, page):
    print(f"search lens={lens} width={width} new={new} {store}", flush=True)
    d = _decoder(gpu_ctx, store, rope, page=page, n_pages=400)
    if stop >= 0:
        d.w["head_bias"][stop] = 6.0
    g = torch.Generator().manual_seed(sum(lens))
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in lens]
    got = [tuple(t.cpu() for t in d.beam(prompts, width, new, stop, pen, temp, graph)) for graph in (False, True, True)]
    for out, total in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(total, got[0][1])
    out, total = got[0]
    # what the pages say of themselves
    p = d.pages
    table, refs, held = p.block_table.cpu(), p.refs.cpu(), [-(-(n + new - 1) // page) for n in lens]
    assert int(p.missing) == 0 and torch.equal(p.lens.cpu(), torch.tensor([n + new - 1 for n in lens]).int().repeat_interleave(width))
    assert torch.equal(torch.bincount(table[table >= 0].flatten(), minlength=p.n_pages).int(), refs)
    assert ((table >= 0).sum(1) == torch.tensor(held).repeat_interleave(width)).all()
    bits = torch.from_numpy(np.unpackbits(p.free_bits.cpu().numpy().view(np.uint8), bitorder="little"))[:p.n_pages].bool()
    assert torch.equal(bits, refs == 0)
    assert (refs > 0).sum() <= sum(n // page + width * (h - n // page) for n, h in zip(lens, held))
    # best first; behind a stop token only stop tokens
    assert (total[:, 1:] <= total[:, :-1]).all()
    if stop >= 0:
        ended = (out == stop).int().cumsum(-1)[..., :-1] > 0
        assert (out[..., 1:][ended] == stop).all() and ended.any()
    want, score = _unshared(d, prompts, width, new, stop, pen, temp)
    assert np.array_equal(out.flatten(0, 1).numpy(), want)
    # a total of up to `new` terms, each a logit's difference and a logarithm in 64 bits, rounded to 32 bits a step
    assert (np.abs(total.flatten().numpy() - score) <= new * 2.0 ** -23 * np.abs(score) + 1e-30).all()


def test_one_beam_is_the_greedy_choice(gpu_ctx):
    d = _decoder(gpu_ctx, "q4", True)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (30, 1, 77, 5)]
    full = lambda v, t: torch.full((4,), v, dtype=t, device="cuda")  # noqa: E731
    par = (full(1.0, torch.float32), full(1, torch.int32), full(1.0, torch.float32), full(1.0, torch.float32))
    want = d.generate(prompts, 25, *par, torch.arange(1, 5, device="cuda"))
    out, total = d.beam(prompts, 1, 25)
    assert torch.equal(out[:, 0], want)
    assert torch.isfinite(total).all() and (total < 0).all()


def test_refusals_of_a_search(gpu_ctx):
    d = _decoder(gpu_ctx, "q4", True, layers=1, n_pages=20)
    ok = [[1] * 40]
    for prompts, width, new, kw in (([[]], 2, 3, {}), ([], 2, 3, {}), (ok, 0, 3, {}), (ok, 33, 3, {}), (ok, 2, 0, {}), ([[VOCAB]], 2, 3, {}),
                                    (ok, 2, 3, dict(stop_token=VOCAB)), (ok, 2, 3, dict(stop_token=-2)), ([[1] * 160] * 2, 2, 16, {}),
                                    (ok, 20, 3, {}), ([[1]] * 129, 32, 1, {})):
        with pytest.raises(ValueError):
            d.beam(prompts, width, new, **kw)
    with pytest.raises(ValueError):      # no room after a search or a refusal
        d.step(torch.zeros(1, dtype=torch.int32, device="cuda"))
    out, total = d.beam(ok, 2, 3)
    assert out.shape == (1, 2, 3) and total.shape == (1, 2) and not math.isnan(float(total.sum()))
    with pytest.raises(ValueError):
        _decoder(gpu_ctx, "q2", True)
