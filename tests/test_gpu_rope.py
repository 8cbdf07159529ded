"""Rotary positions (c4s_rope) against float64.

Bounds: the angle's part of a turn is rounded to float32 (2^-25 of a turn: 2e-7 radians) and its cosine and sine to
within 2 units: each below 3.5e-7; with the product's, the difference's and scale's roundings of 2^-24 each, 6e-7 of
|a| + |b| in all; then half a unit of a bf16 result (a whole one where that crosses a boundary)."""
import pytest
import torch

import batch_util as B
import c4s
import layers_util as L

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
I32 = torch.int32


def _close(got, want, size, dtype):
    err = 6e-7 * size + (L.BF16 * want.abs() if dtype == torch.bfloat16 else 0)
    bad = ~((L.f64(got) - want).abs() <= err)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}"


CASES = [  # new, past, heads, kv_heads, dim, rot, dtype
    ([1] * 5, [0, 1, 700, 63, 9], 20, 20, 64, 64, "bf16"),
    ([1], [1499], 32, 8, 128, 64, "bf16"),
    ([5, 0, 130, 1], [0, 7, 1000, 120000], 4, 2, 128, 128, "bf16"),
    ([3, 64], [200, 0], 12, 12, 80, 20, "bf16"),       # halves of ten
    ([7, 2], [0, 5], 3, 1, 6, 4, "bf16"),
    ([40], [3], 5, 5, 256, 256, "f32"),
    ([9, 30], [90, 1], 4, 4, 64, 16, "f32"),
    ([2, 2], [1, 1], 1, 1, 2, 2, "f32"),
    ([1500], [5], 2, 1, 64, 64, "bf16"),               # a row a workgroup
    ([20], [2 ** 31 - 30], 2, 1, 64, 64, "f32"),
    ([3], [1], 1, 1, 1024, 1024, "bf16"),
    ([3], [5], 2, 1, 7, 4, "bf16"),                    # heads of odd sizes
    ([4], [9], 3, 2, 33, 10, "f32"),
    ([1100], [0], 1, 1, 3, 2, "f32"),
]


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("new,past,heads,kv_heads,dim,rot,dtype", CASES)
def test_rope(gpu_ctx, new, past, heads, kv_heads, dim, rot, dtype, pairs):
    print(f"rope {new} {past} {heads}/{kv_heads} dim={dim} rot={rot} {dtype} pairs={pairs}", flush=True)
    g = torch.Generator().manual_seed(dim + rot)
    rows, t, scale = sum(new), DT[dtype], 1.25
    qkv = torch.randn((rows, heads + 2 * kv_heads, dim), generator=g).to(t)
    freq = c4s.rope_freqs(rot, 10000.0, 8.0, "linear" if rot > 16 else "none")
    lens = torch.tensor([n + p for n, p in zip(new, past)], dtype=I32)
    off = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=I32)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)])
    d = qkv.cuda()
    q, k = d[:, :heads], d[:, heads:heads + kv_heads]
    qo, ko = torch.full_like(d, 7.0)[:, :heads], torch.full((rows, kv_heads, dim), 7.0, dtype=t, device="cuda")
    where = dict(lens=lens.cuda(), rows_off=None if max(new) == min(new) == 1 else off.cuda())
    gpu_ctx.rope(q, k, freq, q_out=qo, k_out=ko, pairs=pairs, scale=scale, **where)
    for x, got in ((qkv[:, :heads], qo), (qkv[:, heads:heads + kv_heads], ko)):
        want, size = B.rope(x, pos, freq, pairs, scale)
        _close(got, want, size, t)
        assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
    # in place, by given positions, and one tensor alone: the same bits; what lies beside is left alone
    gpu_ctx.rope(q, k, freq, pos=pos.to(I32).cuda(), pairs=pairs, scale=scale)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(d[:, heads + kv_heads:].cpu(), qkv[:, heads + kv_heads:])
    alone = qkv.cuda()
    gpu_ctx.rope(None, alone[:, heads:heads + kv_heads], freq, pairs=pairs, scale=scale, **where)
    assert torch.equal(alone[:, heads:heads + kv_heads], ko) and torch.equal(alone[:, :heads].cpu(), qkv[:, :heads])


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_unaligned(gpu_ctx, dtype, pairs):
    """Rows that start anywhere, strides that are odd."""
    g = torch.Generator().manual_seed(1)
    for at, extra in ((1, 3), (3, 2), (4, 0), (8, 8)):
        x = torch.randn((6, 3 * 64 + extra + at), generator=g).to(DT[dtype])
        d = x.cuda()
        q = d[:, at:at + 192].unflatten(1, (3, 64))
        freq = c4s.rope_freqs(64)
        pos = torch.tensor([5, 0, 77, 4000, 1, 2], dtype=I32)
        gpu_ctx.rope(q, None, freq, pos=pos.cuda(), pairs=pairs)
        want, size = B.rope(x[:, at:at + 192].unflatten(1, (3, 64)), pos, freq, pairs, 1.0)
        _close(q, want, size, DT[dtype])
        assert torch.equal(d[:, :at].cpu(), x[:, :at]) and torch.equal(d[:, at + 192:].cpu(), x[:, at + 192:])


def test_rows_of_no_sequence_are_left_alone(gpu_ctx):
    x = torch.ones((10, 1, 64), dtype=torch.bfloat16, device="cuda")
    freq = c4s.rope_freqs(64)
    lens = torch.tensor([3, 1, 2], dtype=I32).cuda()     # the last: more rows than tokens
    off = torch.tensor([2, 4, 4, 7], dtype=I32).cuda()
    gpu_ctx.rope(x, None, freq, lens, off)
    y = x.cpu().float()
    changed = (y != 1).flatten(1).any(1).tolist()
    assert changed == [False, False, True, True, False, False, True, False, False, False]   # row 5: position 0
    x.fill_(1.0)
    gpu_ctx.rope(x, None, freq, pos=torch.tensor([-1, 1, -5] + [0] * 7, dtype=I32).cuda())
    assert (x.cpu() != 1).flatten(1).any(1).tolist() == [False, True] + [False] * 8


def test_turning_back_and_special_values(gpu_ctx):
    """Negated frequencies undo it; infinities and NaN stay in their own pair."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn((50, 4, 64), generator=g).cuda()
    pos = (torch.arange(50) * 997).to(I32).cuda()
    freq = c4s.rope_freqs(64)
    y = x.clone()
    gpu_ctx.rope(y, None, freq, pos=pos)
    assert (y - x).abs().max() > 1
    gpu_ctx.rope(y, None, -freq, pos=pos)
    assert (y - x).abs().max() < 1e-5
    x[7, 2, 3], x[9, 0, 40] = float("nan"), float("inf")
    gpu_ctx.rope(x, None, freq, pos=pos)
    odd = (~torch.isfinite(x)).nonzero().tolist()
    assert odd == [[7, 2, 3], [7, 2, 35], [9, 0, 8], [9, 0, 40]]


def test_in_a_graph_and_on_a_stream(gpu_ctx):
    g = torch.Generator().manual_seed(3)
    q, k = torch.randn((9, 8, 64), generator=g).bfloat16().cuda(), torch.randn((9, 2, 64), generator=g).bfloat16().cuda()
    qo, ko, freq = torch.empty_like(q), torch.empty_like(k), c4s.rope_freqs(64)
    lens = torch.arange(9, dtype=I32).cuda() + 1
    call = lambda: gpu_ctx.rope(q, k, freq, lens, q_out=qo, k_out=ko)  # noqa: E731
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call()
    for step in range(4):
        lens.add_(step * 50)
        call()
        want = qo.clone(), ko.clone()
        qo.zero_(), ko.zero_()
        graph.replay()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    side.wait_stream(torch.cuda.current_stream())
    qo.zero_()
    torch.cuda.synchronize()
    gpu_ctx.rope(q, k, freq, lens, q_out=qo, k_out=ko, stream=side)
    side.synchronize()
    assert torch.equal(qo, want[0])


def test_no_rows_and_refusals(gpu_ctx):
    z = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    freq, lens = c4s.rope_freqs(64), z(2, t=I32)
    gpu_ctx.rope(z(0, 2, 64), z(0, 1, 64), freq, lens, z(3, t=I32))
    gpu_ctx.rope(z(5, 2, 64), None, freq, z(0, t=I32), z(1, t=I32))
    for kw, what in ((dict(freq=c4s.rope_freqs(66)), "rot_dim"), (dict(scale=float("inf")), "scale"),
                     (dict(), "more rows than sequences"), (dict(freq=z(0, t=torch.float64)), "rot_dim")):
        with pytest.raises(c4s.C4SError, match=f"code 1.*{what}"):
            gpu_ctx.rope(z(3, 2, 64), None, **{"freq": freq, "lens": lens, **kw})
    for bad in (lambda: gpu_ctx.rope(z(2, 2, 64), None, freq), lambda: gpu_ctx.rope(None, None, freq, lens)):
        with pytest.raises(ValueError, match="needs"):
            bad()
    x = z(2, 2, 2, 64)
    with pytest.raises(c4s.C4SError, match="code 1.*both strides"):
        gpu_ctx.rope(x[:, 0], None, freq, lens, q_out=x.view(4, 2, 64)[:2])
    for bad in (lambda: gpu_ctx.rope(z(2, 2, 64), z(3, 2, 64), freq, lens), lambda: gpu_ctx.rope(z(2, 2, 64), z(2, 2, 64, t=torch.float32), freq, lens),
                lambda: gpu_ctx.rope(z(2, 2, 64), None, freq.float(), lens), lambda: gpu_ctx.rope(z(2, 2, 64), None, freq, lens, z(2, t=I32)),
                lambda: gpu_ctx.rope(z(2, 2, 64), None, freq, lens, q_out=z(2, 3, 64)), lambda: gpu_ctx.rope(z(2, 2, 64, t=torch.float16), None, freq, lens),
                lambda: gpu_ctx.rope(z(2, 2, 64), None, freq, pos=z(3, t=I32))):
        with pytest.raises(ValueError):
            bad()
    torch.cuda.synchronize()
