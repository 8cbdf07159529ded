"""The decoder built from the layer's operators (c4s_decode.py): its hidden rows against the same decoder in
float64, prompts against tokens one by one, and graph replays against eager steps."""
import pytest
import torch

import c4s_decode as D
import layers_util as L

pytestmark = pytest.mark.gpu

VOCAB = 515


def _reference(w, ids, heads, kv_heads):
    """Residual rows of one sequence after the last layer, float64 on the CPU."""
    x = L.f64(w["tokens"][ids]) + L.f64(w["positions"][:len(ids)])
    n, hd = len(ids), x.shape[1] // heads
    ln = lambda v, p: L.norm(v, False, 1e-5, *p)  # noqa: E731
    mask = torch.full((n, n), float("-inf"), dtype=torch.float64).triu(1)
    for l in w["layers"]:
        qkv = (ln(x, l["norm1"]) @ L.f64(l["qkv"]).t() + L.f64(l["qkv_bias"])).view(n, heads + 2 * kv_heads, hd)
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        s = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) * hd ** -0.5 + mask, -1)
        a = torch.einsum("hij,jhd->ihd", s, v).reshape(n, -1)
        x = x + a @ L.f64(l["out"]).t() + L.f64(l["out_bias"])
        m = L.gelu(ln(x, l["norm2"]) @ L.f64(l["up"]).t() + L.f64(l["up_bias"]))
        x = x + m @ L.f64(l["down"]).t() + L.f64(l["down_bias"])
    return x


def _decoder(ctx, q8=False, heads=8, kv_heads=4, layers=3):
    w = D.random_weights(layers, heads * 64, heads, kv_heads, VOCAB, 400, seed=7)
    for l in w["layers"]:   # blocks that weigh as much as the embeddings
        for k in ("qkv", "out", "up", "down"):
            l[k] = (l[k].float() * 3).bfloat16()
    return D.Decoder(ctx, w, heads, kv_heads, 200, q8_cache=q8)


# bf16 roundings of 2^-9 at most: five a block (norm, products, weights), six blocks and the result, independent:
# sqrt(31) 2^-9 = 1.1 % of the row's length if all of it went through every one. Eight-bit keys and values: half a
# step of max / 127, with the maximum of 64 normal numbers below 4 deviations, uniform: 4 / 127 / sqrt(12) = 0.9 %,
# twice a layer, three layers: 2.3 %.
BOUND = {False: 0.011, True: 0.026}


@pytest.mark.parametrize("q8", [False, True])
def test_prompts_and_steps_against_float64(gpu_ctx, q8):
    d = _decoder(gpu_ctx, q8)
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randint(0, VOCAB, (n,), generator=g) for n in (90, 17, 213)]
    want = [_reference(d.w, s, d.heads, d.kv_heads) for s in seqs]
    for cut in (0, 1, 6):   # the last `cut` tokens one by one
        h = d.begin([s[:len(s) - cut] for s in seqs], cut + 1)
        for i in range(cut, 0, -1):
            h = d.step(torch.stack([s[-i] for s in seqs]).cuda())
        assert d.lens.tolist() == [len(s) for s in seqs]
        for got, x in zip(h, want):
            err = (L.f64(got) - x[-1]).norm() / x[-1].norm()
            print(f"q8={q8} cut={cut}: {err:.4f}", flush=True)
            assert err <= BOUND[q8]


def test_generate_with_a_graph_and_without(gpu_ctx):
    d = _decoder(gpu_ctx, q8=True)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (30, 1, 77, 5)]
    full = lambda v, t: torch.full((4,), v, dtype=t, device="cuda")  # noqa: E731
    par = (full(0.9, torch.float32), full(40, torch.int32), full(0.9, torch.float32), full(1.2, torch.float32))
    runs, states = [], []
    for graph in (False, True, True):
        rng = torch.arange(1, 5, device="cuda") * 0x100000001B3
        runs.append(d.generate(prompts, 40, *par, rng, graph=graph))
        states.append(rng)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    assert torch.equal(states[0], states[1]) and torch.equal(states[0], states[2])
    assert ((runs[0] >= 0) & (runs[0] < VOCAB)).all() and len(runs[0].unique()) > 20


def test_refusals_of_the_decoder(gpu_ctx):
    d = _decoder(gpu_ctx, layers=1)
    for prompts, new in (([[]], 3), ([[1] * 399], 2), ([[1] * 300] * 12, 50)):
        with pytest.raises(ValueError):
            d.begin(prompts, new)
