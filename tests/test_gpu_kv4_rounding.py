"""How often attention over 4-bit pages rounds: weights enter as pairs of bf16 in every kernel, single tokens' and
prompts', so that what is left is the result's own rounding. The codes' values are bf16's, and exact.

Bounds: those of test_gpu_attn_rounding.py's pairs. Weights to 2^-17 of themselves, scores and sums in float32: below 1e-4 of
sum w |v|; as a root mean square over a whole result less than a hundredth of the result's own rounding, where weights rounded
once add one of its own kind (1.05 to 1.41 times)."""
import pytest
import torch

import batch_util as B
import layers_util as L
from test_gpu_attn_rounding import _ratio
from test_gpu_kv4 import ATTN, PROMPTS
from test_gpu_layers import _check_attn, _close, _run_attn

pytestmark = pytest.mark.gpu


def _many(new, heads, kv_heads, dim):
    """Whether the prompts' kernel has them: by tiles of 16 (row, query head) pairs of a sequence and key head, and all of them."""
    tiles = -(-max(new) * (heads // kv_heads) // 16)
    return tiles > (3 if dim <= 128 else 1) and tiles * kv_heads * len(new) > (1500 if dim <= 128 else 1100)


WIDE = [([70, 140], [7, 120], 64, 64, 256, 16), ([61, 17, 40], [64, 1000, 0], 96, 24, 192, 256)]   # of heads over 128
CASES = [c for c in ATTN if sum(c[0]) * c[2] * c[4] >= 400] + PROMPTS + WIDE


def test_the_cases_have_prompts_of_every_kernel():
    assert {64 * 2 ** ((c[4] > 64) + (c[4] > 128)) for c in CASES if _many(c[0], *c[2:5])} == {64, 128, 256}


@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page", CASES)
def test_pairs(gpu_ctx, new, past, heads, kv_heads, dim, page):
    cache = B.Cache4([n + p for n, p in zip(new, past)], kv_heads, dim, page, seed=dim + page, junk=True)
    q, out, _ = _run_attn(gpu_ctx, cache, new, heads)
    want, _, mag, _ = L.attn(cache, q, new, heads, dim ** -0.5)
    r = _ratio(out, want)
    print(f"attn4 new={new} past={past} heads={heads}/{kv_heads} dim={dim} page={page}: {r:.4f}", flush=True)
    _close(out, want, 1e-4 * mag)
    assert r <= 1.01


def test_padding_and_missing_pages_with_wide_heads(gpu_ctx):
    """Prompts of heads of 256, padded in front past all of some rows, pages that are not there; what is not seen is not finite."""
    new, past, first, heads = [70, 140, 20], [7, 120, 0], [40, 131, 2 ** 31 - 1], 48
    assert _many(new, heads, heads, 256)
    cache = B.Cache4([n + p for n, p in zip(new, past)], heads, 256, 16, seed=5, junk=True)
    for b, f in enumerate(first):
        for p in range(min(f, cache.lens[b])):
            cache.spoil("k", b, p)
            cache.spoil("v", b, p)
    cache.table[1, 10:12] = torch.tensor([-1, cache.n_pages + 3])
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, first=first, spread=0.7)
    empty = torch.isinf(L.attn(cache, q, new, heads, 0.0625, first)[1])
    assert empty.any() and (out.cpu()[empty] == 0).all()
    _check_attn(cache, q, out, lse, new, heads, first=first)


@pytest.mark.parametrize("byte", [47, 221])
@pytest.mark.parametrize("new,past,heads,kv_heads,dim", [([1, 1], [300, 20], 3, 3, 64), ([1, 1], [300, 20], 12, 3, 128), ([6, 1], [300, 20], 5, 5, 256),
                                                         ([150, 80], [40, 3], 80, 80, 64)])
def test_values_as_small_and_as_large_as_attention_has_them(gpu_ctx, byte, new, past, heads, kv_heads, dim):
    """All scales 2^-80, or 2^94: values up to 2^96.6."""
    cache = B.Cache4([n + p for n, p in zip(new, past)], kv_heads, dim, 16, seed=dim, junk=True)
    cache.t["v_scale"][cache.t["v_scale"] != 255] = byte
    q, out, lse = _run_attn(gpu_ctx, cache, new, heads, spread=0.7)
    _check_attn(cache, q, out, lse, new, heads)
