"""How exact a beam step's totals are (c4s_beam_step): the sum of exponentials against float64.

Bound of log sum exp z, as the header has it. With d = z - max: a difference's rounding and a product's, 2^-24 each, and the
rounded log2 e, 2^-26, are errors of the exponent of at most 2^-22.8 |d|; the exponential itself is good to 2^-23; sixteen of them are
added in four float32 additions on each one's way, 2^-24 each, all others in float64. Together below 2^-22 (1.5 + |d|) of an
exponential, so of the sum and its logarithm 2^-22 (1.5 + the mean of |d|, weighted by exp d). The total is then rounded to float32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _log_sum(z):
    """(log sum exp, bound of its error) of rows in float64."""
    top = z.amax(1, keepdim=True)
    w = torch.exp(z - top)
    s = w.sum(1)
    return top[:, 0] + torch.log(s), 2.0 ** -22 * (1.5 + ((top - z) * w).sum(1) / s)


def _step(ctx, logits, width, score):
    rows = len(logits)
    out, parent, token = torch.empty_like(score), torch.empty(rows, dtype=I32, device="cuda"), torch.empty(rows, dtype=I32, device="cuda")
    ctx.beam_step(logits, width, score, out, parent, token)
    return out.cpu().double(), parent.cpu().long(), token.cpu().long()


def _check(ctx, row, groups, width):
    """Every row of the call is `row` (float32 [vocab]); scores that leave totals near 0, where float32 rounds little."""
    z = row.double()[None]
    lse, err = _log_sum(z)
    rows = groups * width
    score = torch.full((rows,), float(lse - row.max()), device="cuda")
    score += torch.arange(rows, device="cuda") % width * 1e-3
    out, parent, token = _step(ctx, row.cuda().expand(rows, -1).contiguous(), width, score)
    want = score.cpu().double().view(-1, width).gather(1, parent.view(-1, width)).flatten() + (row.double()[token] - lse)
    off = (out - want).abs()
    print(f"{groups} x {width} x {len(row)}: {off.max():.2e}, bound {err.item():.2e}", flush=True)
    assert (off <= err + 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("peak", [0, 7, 31])
def test_many_alike_beside_a_peak(gpu_ctx, peak):
    """One slice a row, 32 chunks of 16 a lane: one of them holds ones, all others the same small numbers, whose additions
    one after another would all round the same way."""
    row = torch.full((32000,), -3.464)
    row[1024 * peak:1024 * (peak + 1)] = 0.0
    _check(gpu_ctx, row, 1024, 4)


def test_maxima_that_rise_a_little(gpu_ctx):
    """Every chunk has a new maximum: what was summed before is scaled every time."""
    for step in (1.5 * 2.0 ** -25, 1e-3, 0.7):
        row = (torch.arange(32768) // 1024).double().mul(step).float() + 1.0 if step > 1e-6 else 2.0 ** -3 + (torch.arange(32768) // 1024 * step)
        _check(gpu_ctx, row.float(), 1024, 4)


@pytest.mark.parametrize("groups,width,vocab", [(1, 2, 100), (1, 4, 8194), (2, 3, 151936), (300, 4, 20001), (1, 1, 1 << 20)])
def test_random_rows(gpu_ctx, groups, width, vocab):
    g = torch.Generator().manual_seed(vocab)
    for size in (0.1, 3.0, 30.0):
        _check(gpu_ctx, torch.randn(vocab, generator=g) * size, groups, width)


def test_a_wide_flat_row_beside_one_peak(gpu_ctx):
    """The largest vocabulary: half of the sum is in a million numbers far below the largest."""
    row = torch.full((1 << 20,), -13.8155)
    row[777777] = 0.0
    _check(gpu_ctx, row, 2, 2)
    _check(gpu_ctx, row, 64, 2)


def test_near_ties_of_two_beams(gpu_ctx):
    """Totals that differ by little more than both sums' bounds come in their order, however many rows the call has."""
    flat = torch.full((32000,), -3.464)
    flat[:1024] = 0.0
    peaked = torch.full((32000,), -60.0)
    peaked[4], peaked[5] = 1.0, 0.5
    (a, ea), (b, eb) = _log_sum(flat.double()[None]), _log_sum(peaked.double()[None])
    gap = 1.5 * float(ea + eb)
    for groups in (1, 30, 1024):
        for sign in (1, -1):
            # the second row's best total is 0 but for its score's rounding, the first's lies a gap above or below it
            score = torch.tensor([float(a) + sign * gap, float(b) - 1.0], dtype=torch.float32).repeat(groups)
            best = torch.stack([score[0].double() - a[0], score[1].double() + 1.0 - b[0]])
            if (best[0] - best[1]) * sign < float(ea + eb):    # float32 scores are 5e-7 apart there
                score[0::2] = torch.nextafter(score[0], torch.tensor(sign * torch.inf))
                best[0] = score[0].double() - a[0]
            assert float(ea + eb) < (best[0] - best[1]) * sign < 4e-6
            _, parent, token = _step(gpu_ctx, torch.stack([flat, peaked]).cuda().repeat(groups, 1), 2, score.cuda())
            assert parent.view(-1, 2)[:, 0].tolist() == [0 if sign > 0 else 1] * groups
            assert token.view(-1, 2)[:, 0].tolist() == [0 if sign > 0 else 4] * groups
