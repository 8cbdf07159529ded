"""How often attention rounds (c4s_attn): weights as pairs of bf16 for few rows and for 8-bit pages, so that what is
left is the result's own rounding; rounded once for prompts over bf16 pages alone.

Bounds. Pairs hold a weight to 2^-17 of itself, scores and sums are float32: together below 1e-4 of sum w |v| (as in
test_gpu_layers.py, without its allowance for weights rounded once). As a root mean square over a whole result they
add to its own rounding, about 2^-9 / sqrt(3) of each value, less than a hundredth of it: both are independent,
and 1e-5 of a value is far more than pairs and scores of this size leave. Weights rounded once have errors of
the result's own kind: each of up to sqrt(sum w^2 v^2), as large as the result itself where the values' signs are
random: sqrt(2) times the rounding alone, and no less than 1.05 where the weights are not exact."""
import pytest
import torch

import layers_util as L
from test_gpu_layers import PROMPTS as FEW, _close, _run_attn
from test_gpu_layers_many import PROMPTS as MANY, _fills

pytestmark = pytest.mark.gpu


def _case(ctx, new, past, heads, kv_heads, dim, page, q8, **k):
    cache = L.Cache([n + p for n, p in zip(new, past)], kv_heads, dim, page, q8, seed=dim + page, junk=float("nan"))
    q, out, lse = _run_attn(ctx, cache, new, heads, **k)
    want, wlse, mag, _ = L.attn(cache, q, new, heads, dim ** -0.5)
    return out, want, mag


def _ratio(out, want):
    """The result's error by the error of rounding the exact one, root mean squares."""
    rounded = want.to(torch.bfloat16).double()
    return ((L.f64(out) - want).square().mean().sqrt() / (rounded - want).square().mean().sqrt()).item()


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,q8", FEW + [c for c in MANY if c[-1]])
def test_pairs(gpu_ctx, new, past, heads, kv_heads, dim, page, q8):
    many = _fills(new, heads, kv_heads, len(new), q8, dim)
    assert q8 or not many
    out, want, mag = _case(gpu_ctx, new, past, heads, kv_heads, dim, page, q8)
    r = _ratio(out, want)
    print(f"attn new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page} q8={q8} many={many}: {r:.4f}", flush=True)
    _close(out, want, 1e-4 * mag)
    assert r <= 1.01


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page,q8", [c for c in MANY if not c[-1]])
def test_weights_rounded_once(gpu_ctx, new, past, heads, kv_heads, dim, page, q8):
    assert _fills(new, heads, kv_heads, len(new), q8, dim)
    out, want, _ = _case(gpu_ctx, new, past, heads, kv_heads, dim, page, q8)
    r = _ratio(out, want)
    print(f"attn new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page}: {r:.4f}", flush=True)
    assert r <= 2 ** 0.5 + 0.02
