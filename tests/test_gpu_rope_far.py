"""Rotary positions whose angles are hundreds of millions of turns and more (c4s_rope).

The product of position and frequency and the division by 2 pi keep what 64 bits lose, so far positions have the bound of near ones:
the rest of a turn is rounded to float32, 2^-26 of a turn or 1e-7 radians; its cosine and sine are good to two units, 1.2e-7; scale,
a product and the difference round by 2^-24 each: 4e-7 of |a| + |b|. The frequencies have few bits, so that position * frequency is exact
in float64, and its cosine and sine are the C library's."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FREQ = [1.0, 0.75, 3.0, 1000.0, -1.0, 2.0 ** -20, 2.0 ** 15 + 1, 0.0]
POS = [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 12345, 1234567890, 987654321, 10 ** 6, 999999, 355, 1, 0]


@pytest.mark.parametrize("pairs", [False, True])
def test_far_positions(gpu_ctx, pairs):
    g = torch.Generator().manual_seed(1)
    pos = POS + [2 ** 31 - 1 - 7919 * i for i in range(500)]
    n, half = len(pos), len(FREQ)
    x = torch.randn((n, 2, 2 * half + 4), generator=g)
    d = x.cuda()
    gpu_ctx.rope(d, None, torch.tensor(FREQ, dtype=torch.float64).cuda(), pos=torch.tensor(pos, dtype=torch.int32).cuda(), pairs=pairs)
    got = d.cpu().double()
    angle = [[p * f for f in FREQ] for p in pos]
    cos, sin = (torch.tensor([[f(a) for a in row] for row in angle], dtype=torch.float64)[:, None] for f in (math.cos, math.sin))
    at = torch.arange(2 * half).view(-1, 2).t() if pairs else torch.arange(2 * half).view(2, -1)
    a, b = x[..., at[0]].double(), x[..., at[1]].double()
    for part, want in ((at[0], a * cos - b * sin), (at[1], a * sin + b * cos)):
        off = (got[..., part] - want).abs() / (a.abs() + b.abs())
        print([f"{v:.1e}" for v in off.amax((0, 1)).tolist()], flush=True)
        assert (off <= 4e-7).all()
    assert torch.equal(got[..., 2 * half:], x[..., 2 * half:].double())
