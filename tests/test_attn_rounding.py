"""The bounds of test_gpu_attn_rounding.py told apart without a GPU: attention in float64 with its weights (for 8-bit
pages times their values' scales) rounded to bf16 once, and to pairs of bf16."""
import pytest
import torch

import layers_util as L


def _bf16(x):
    return x.to(torch.bfloat16).double()


@pytest.mark.parametrize("n,dim,q8", [(130, 64, False), (130, 64, True), (40, 128, True), (300, 16, True)])
def test_a_lost_low_half_shows(n, dim, q8):
    cache = L.Cache([n], 1, dim, 16, q8, seed=n)
    q = (torch.randn((n, 1, dim), generator=torch.Generator().manual_seed(1)) * 1.5).to(torch.bfloat16)
    want = L.attn(cache, q, [n], 1, dim ** -0.5)[0][:, 0]
    k, _ = cache.rows("k", 0, n)
    v, _ = cache.rows("v", 0, n)
    scale = torch.ones(n, dtype=torch.float64)
    if q8:
        scale = torch.stack([cache.t["v_scale"][cache.table[0, p // 16], 0, p % 16] for p in range(n)]).double()
    z = (L.f64(q)[:, 0] @ k[:, 0].t() * dim ** -0.5).masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf)
    w = torch.exp(z - z.amax(1, keepdim=True))
    x = w * scale
    rounded = _bf16(want) - want
    for parts, test in ((_bf16(x), lambda r: r > 1.05), (_bf16(x) + _bf16(x - _bf16(x)), lambda r: r <= 1.01)):
        out = _bf16(parts @ (v[:, 0] / scale[:, None]) / w.sum(1, keepdim=True))
        r = ((out - want).square().mean().sqrt() / rounded.square().mean().sqrt()).item()
        print(f"{n} x {dim}, q8={q8}: {r:.4f}")
        assert test(r)
