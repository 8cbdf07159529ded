"""Equal totals of different logits (c4s_beam_step): tokens whose logits differ by less than a total in 64 bits can hold. The
lowest (beam, token) comes first, as with equal logits, however a row is cut."""
import numpy as np
import pytest
import torch

import batch_util as B
from test_gpu_beam import _run

pytestmark = pytest.mark.gpu
LOW = np.finfo(np.float32).min


def _same(ctx, z, width, score, **k):
    host = z.float().cpu().numpy() if isinstance(z, torch.Tensor) else z
    got = _run(ctx, z, width, score, **k)
    want = B.beams(host, width, score, k.get("done"), k.get("stop", -1), k.get("temp"), k.get("pen"), k.get("bits"))
    assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()
    assert np.array_equal(np.isinf(got[2]), np.isinf(want[2])) and np.array_equal(np.sign(got[2]), np.sign(want[2]))
    fine = np.isfinite(want[2])
    # a log sum's bound for these rows, and float32's rounding
    assert (np.abs(got[2] - want[2])[fine] <= 2 ** -20 + 2.0 ** -23 * np.abs(want[2][fine])).all()
    return want


SIZES = [(2, 40), (4, 1000), (1, 5000), (3, 8194), (8, 50001), (32, 9000), (32, 40000)]


@pytest.mark.parametrize("width,vocab", SIZES)
@pytest.mark.parametrize("low", [-1e30, LOW, np.inf])
def test_scores_that_leave_nothing_of_the_logits(gpu_ctx, width, vocab, low):
    """Beams that are masked by a finite score (and one of +inf): all their tokens have one total."""
    print(f"{width} x {vocab} {low}", flush=True)
    r = np.random.default_rng(vocab)
    z = (r.standard_normal((3 * width, vocab)) * 3).astype(np.float32)
    z[:, :vocab // 2] -= 5                                   # the highest logits are not the lowest tokens
    all_low = np.full(3 * width, low, np.float32)
    want = _same(gpu_ctx, z, width, all_low)
    assert want[1][:width].tolist() == list(range(width)) and not want[0].any()
    _same(gpu_ctx, torch.from_numpy(z).to(torch.bfloat16).cuda(), width, all_low)
    first = np.where(np.arange(3 * width) % width == 0, -1.5, low).astype(np.float32)
    few = z.copy()
    few[::width] = -np.inf                                   # a beam that is there, with one token left, or two
    few[::width, vocab - 1] = 2.0
    few[width, 5] = 1.0
    _same(gpu_ctx, few, width, first)
    done = np.arange(3 * width) % 3 == 1
    _same(gpu_ctx, few, width, first, done=done, stop=vocab - 3)
    _same(gpu_ctx, few, width, first, done=done, stop=1, temp=np.full(3 * width, 0.8, np.float32), pen=np.full(3 * width, 1.3, np.float32),
          bits=r.random(z.shape) < 0.3)


@pytest.mark.parametrize("width,vocab", SIZES)
def test_logits_that_vanish_beside_the_largest(gpu_ctx, width, vocab):
    """One token far above the others, of which some differ by less than its last bit; zeros of both signs among them."""
    r = np.random.default_rng(width)
    z = np.full((2 * width, vocab), -np.inf, np.float32)
    for row in z:
        at = r.choice(vocab, min(vocab, 40 + vocab // 20), replace=False)
        row[at] = r.choice(np.array([1e-20, -1e-20, 3e-25, 0.0, -0.0, 1e-45, -1e-45], np.float32), len(at))
        row[at[0]] = 30.0
    score = np.where(np.arange(2 * width) % width == 0, -r.random(2 * width), -100).astype(np.float32)
    want = _same(gpu_ctx, z, width, score)
    assert (want[0] == 0).all() and (want[2].reshape(2, width)[:, 1:] < -29).all()   # the largest, and those that tie
    # beams alike (of others the log sums, which differ by e^-30, would decide, and they are good to 2^-22)
    _same(gpu_ctx, np.tile(z[:1], (2 * width, 1)), width, np.zeros(2 * width, np.float32))
    _same(gpu_ctx, torch.from_numpy(z).to(torch.bfloat16).cuda(), width, score)
    every = np.where(np.isneginf(z), np.float32(-1e-22), z)   # nothing masked: most of the row has one total
    _same(gpu_ctx, every, width, score)


def test_as_many_rows_as_it_takes_to_cut_them_otherwise(gpu_ctx):
    z = (np.random.default_rng(3).standard_normal((4, 9000)) * 3).astype(np.float32)
    score = np.array([-1e30, -1e30, 0, LOW], np.float32)
    z[2, 1:] = -np.inf
    for times in (1, 60, 1000):
        want = _same(gpu_ctx, torch.from_numpy(z).cuda().repeat(times, 1) if times > 60 else np.tile(z, (times, 1)), 4, np.tile(score, times))
        assert want[0][:4].tolist() == [2, 0, 0, 0] and want[1][:4].tolist() == [0, 0, 1, 2]


def test_equal_logits_in_lists_too_long_to_rank_at_once(gpu_ctx):
    """Flat rows, and rows of two values, cut into many slices: every place of every list reaches the bound."""
    for width, vocab in ((32, 60000), (32, 200000), (16, 300000)):
        z = np.zeros((width, vocab), np.float32)
        _same(gpu_ctx, z, width, np.zeros(width, np.float32))
        _same(gpu_ctx, z, width, np.full(width, -1e30, np.float32))
        z[:, ::3] = 1e-22
        _same(gpu_ctx, z, width, np.zeros(width, np.float32))
        z[:, ::3] = np.float32(2.0 ** -20)
        _same(gpu_ctx, z, width, np.zeros(width, np.float32))
