"""Beam search's step (c4s_beam_step) against a sort of all candidates in float64: parents, tokens, states exactly,
totals to float32's rounding and the sum of exponentials' (2^-20 absolute: each is off by 2^-22 relative at most)."""
import math

import numpy as np
import pytest
import torch

import batch_util as B
import c4s

pytestmark = pytest.mark.gpu
I32, F32, U8 = torch.int32, torch.float32, torch.uint8


def _run(ctx, z, width, score, stream=None, inplace=False, **k):
    """One call on host arrays; (parent, token, total, done, bits, states)."""
    rows, vocab = z.shape
    d = lambda x, t=None: None if x is None else torch.as_tensor(x).to(t or torch.as_tensor(x).dtype).cuda()  # noqa: E731
    logits = z if isinstance(z, torch.Tensor) else d(z)
    sc, done, bits = d(score, F32), d(k.get("done"), U8), None if k.get("bits") is None else B.pack_bits(k["bits"]).cuda()
    empty = lambda x: None if x is None else (x if inplace else torch.full_like(x, 99))  # noqa: E731
    out_sc, out_bits = empty(sc), empty(bits)
    out_done = empty(done) if done is not None else torch.full((rows,), 99, dtype=U8, device="cuda")
    parent, token = (torch.full((rows,), -9, dtype=I32, device="cuda") for _ in "pt")
    states = [(s, s if inplace else torch.full_like(s, 99)) for s in (d(x) for x in k.get("states", []))]
    ctx.beam_step(logits, width, sc, out_sc, parent, token, done=done, out_done=out_done, stop_token=k.get("stop", -1),
                  temp=d(k.get("temp"), F32), pen=d(k.get("pen"), F32), hist_bits=bits, out_hist_bits=out_bits,
                  states=states, stream=stream)
    torch.cuda.synchronize()
    return (parent.cpu().numpy(), token.cpu().numpy(), out_sc.cpu().numpy(), out_done.cpu().numpy(),
            None if bits is None else out_bits.cpu(), [s[1].cpu() for s in states])


def _check(ctx, z, width, score, inplace=False, **k):
    host = z.float().cpu().numpy() if isinstance(z, torch.Tensor) else z
    got = _run(ctx, z, width, score, inplace=inplace, **k)
    want = B.beams(host, width, score, k.get("done"), k.get("stop", -1), k.get("temp"), k.get("pen"), k.get("bits"))
    assert got[0].tolist() == want[0].tolist() and got[1].tolist() == want[1].tolist()
    assert got[3].astype(bool).tolist() == want[3].tolist() and set(got[3].tolist()) <= {0, 1}
    inf = np.isinf(want[2])
    assert (np.isneginf(got[2]) == inf).all()
    assert (np.abs(got[2][~inf] - want[2][~inf]) <= 2 ** -20 + 2 ** -23 * np.abs(want[2][~inf])).all()
    if want[4] is not None:
        assert torch.equal(got[4], B.pack_bits(want[4]))
    at = np.arange(len(host)) // width * width + want[0]
    for s, x in zip(k.get("states", []), got[5]):
        assert torch.equal(x, torch.as_tensor(s)[torch.as_tensor(at)])
    return got


CASES = [  # groups, width, vocab, bf16
    (1, 1, 1, False), (2, 3, 2, False), (1, 32, 5, True), (3, 4, 31, False), (1, 3, 8194, False), (64, 4, 8194, False),
    (5, 5, 1023, True), (5, 5, 1025, False), (2, 8, 50001, True), (1, 32, 151936, False), (300, 2, 700, True),
    (700, 6, 64, False), (1, 16, 1048576, True), (33, 1, 12289, True),
]


@pytest.mark.parametrize("groups,width,vocab,bf16", CASES)
def test_beams(gpu_ctx, groups, width, vocab, bf16):
    print(f"beams {groups} x {width} x {vocab} bf16={bf16}", flush=True)
    r = np.random.default_rng(vocab + width)
    rows, stop = groups * width, vocab // 2
    z = torch.from_numpy((r.standard_normal((rows, vocab)) * 3).astype(np.float32)).to(torch.bfloat16 if bf16 else F32).cuda()
    score = (r.standard_normal(rows) * 0.7 - 20).astype(np.float32)
    first = np.where(np.arange(rows) % width == 0, 0, -np.inf).astype(np.float32)
    done = (r.random(rows) < 0.3).astype(np.uint8)
    bits = r.random((rows, vocab)) < 0.1
    pen, temp = r.choice([1.0, 10.0, 1.3], rows).astype(np.float32), r.choice([1.0, 0.8, 0.0, -1.0], rows).astype(np.float32)
    tokens, words = r.integers(0, 9999, (rows, 37)).astype(np.int32), r.standard_normal((rows, 700)).astype(np.float32)
    _check(gpu_ctx, z, width, score)
    _check(gpu_ctx, z, width, first, stop=stop, states=[tokens])
    _check(gpu_ctx, z, width, score, done=done, stop=stop, temp=temp, pen=pen, bits=bits, states=[tokens, words])
    _check(gpu_ctx, z, width, score, done=done, stop=stop, temp=temp, pen=pen, bits=bits, states=[tokens, words], inplace=True)


def test_ties(gpu_ctx):
    """Equal totals go to the lowest (beam, token): constant rows, rows of few values, equal beams."""
    r = np.random.default_rng(5)
    for width, vocab in ((4, 40), (3, 5000), (32, 9000), (8, 8)):
        print(f"ties {width} x {vocab}", flush=True)
        flat = np.zeros((2 * width, vocab), np.float32)
        few = np.tile(r.integers(0, 3, (1, vocab)).astype(np.float32), (2 * width, 1))
        for z in (flat, few, -few):
            got = _check(gpu_ctx, z, width, np.zeros(2 * width, np.float32))
            assert (np.diff(got[0][:width] * vocab + got[1][:width]) > 0).all() or z is few
    # a row that rises, so that every value beats the ones before, and one that falls
    up = np.arange(4 * 6000, dtype=np.float32).reshape(4, 6000) * 0.001
    _check(gpu_ctx, up, 4, np.zeros(4, np.float32))
    _check(gpu_ctx, -up, 4, np.zeros(4, np.float32))
    # all the best in one lane's values: tokens 0-3, 256-259 ...
    z = np.full((1, 4096), -5.0, np.float32)
    z[0, [256 * i + j for i in range(16) for j in range(4)]] = np.arange(64)
    for width in (1,):
        _check(gpu_ctx, z, width, np.zeros(1, np.float32))
    _check(gpu_ctx, np.tile(z, (32, 1)), 32, np.concatenate([[0], np.full(31, -40)]).astype(np.float32))


def test_infinities(gpu_ctx):
    """Masked tokens and rows, beams that are not there yet, all of them done."""
    z = np.random.default_rng(6).standard_normal((8, 300)).astype(np.float32)
    z[0, 5:] = -np.inf           # five tokens left
    z[1] = -np.inf               # none
    z[2, ::2] = -np.inf
    score = np.array([-1, -2, -np.inf, -3, 0, -np.inf, -np.inf, -np.inf], np.float32)
    _check(gpu_ctx, z, 4, score)
    _check(gpu_ctx, z, 8, score)
    _check(gpu_ctx, z, 4, np.full(8, -np.inf, np.float32))
    _check(gpu_ctx, z, 4, score, done=np.array([0, 1, 1, 0] * 2), stop=7)
    _check(gpu_ctx, z, 4, score, done=np.ones(8), stop=299)
    got = _run(gpu_ctx, np.full((2, 3), -np.inf, np.float32), 2, np.zeros(2, np.float32))
    assert got[0].tolist() == [0, 0] and got[1].tolist() == [0, 1] and np.isneginf(got[2]).all()
    low = np.full((4, 5000), np.finfo(np.float32).min, np.float32)    # masked by the type's lowest value: a row alone, and whole rows
    low[0, 70], low[1, ::1700] = 2.0, -3.0
    got = _check(gpu_ctx, low, 4, np.array([-1, -2, -30, -0.5], np.float32))
    assert got[0].tolist() == [0, 1, 1, 1]
    _check(gpu_ctx, torch.from_numpy(low).to(torch.bfloat16).cuda(), 2, np.array([-1, -2, -30, -0.5], np.float32))
    _check(gpu_ctx, -low, 4, np.array([-1, -2, -30, -0.5], np.float32))
    one = np.full((3, 40), -np.inf, np.float32)
    one[:, 11] = 4.0             # log-probability 0
    got = _check(gpu_ctx, one, 3, np.array([-1, -2, -3], np.float32), stop=11)
    assert got[2].tolist() == [-1, -2, -3] and got[3].all()


@pytest.mark.parametrize("vocab", [300, 9000])
def test_what_is_not_a_number(gpu_ctx, vocab):
    """Rows with NaN or +inf anywhere, alone or beside masked tokens, and such scores: no total but -inf."""
    r = np.random.default_rng(9)
    for bad in (math.nan, -math.nan, math.inf):
        for at in (0, 17, vocab - 1):
            z = r.standard_normal((12, vocab)).astype(np.float32)
            z[1, at] = z[6, at] = bad
            z[4] = -np.inf
            z[4, at] = bad                # beside nothing but masked tokens
            z[8:] = bad                   # nothing else in the group
            score = r.standard_normal(12).astype(np.float32)
            _check(gpu_ctx, z, 4, score)
            _check(gpu_ctx, torch.from_numpy(z).to(torch.bfloat16).cuda(), 3, score)
            _check(gpu_ctx, z, 4, score, done=np.arange(12) % 3 == 0, stop=5)
            score[5] = score[8] = math.nan
            _check(gpu_ctx, z, 4, score)


def test_strides_and_alignment(gpu_ctx):
    """Rows that start anywhere, wider than the vocabulary; states with strides; what lies behind is left alone."""
    r = np.random.default_rng(7)
    for t, at, wide in ((F32, 1, 1003), (torch.bfloat16, 1, 1003), (torch.bfloat16, 3, 1001), (F32, 0, 1000)):
        z = torch.from_numpy(r.standard_normal((6, wide + at)).astype(np.float32)).to(t).cuda()
        z[:, at + 999:] = 50.0
        _check(gpu_ctx, z[:, at:at + 999], 3, r.standard_normal(6).astype(np.float32))
    src, dst = torch.arange(6 * 50, dtype=I32, device="cuda").view(6, 50), torch.full((6, 40), -1, dtype=I32, device="cuda")
    z, score = torch.randn((6, 100), device="cuda"), torch.zeros(6, device="cuda")
    parent, token = (torch.empty(6, dtype=I32, device="cuda") for _ in "pt")
    gpu_ctx.beam_step(z, 2, score, torch.empty_like(score), parent, token, states=[(src[:, 3:20], dst[:, 5:22])])
    at = (torch.arange(6) // 2 * 2 + parent.cpu()).cuda()
    assert torch.equal(dst[:, 5:22], src[at.long(), 3:20]) and (dst[:, :5] == -1).all() and (dst[:, 22:] == -1).all()


def test_in_a_graph_and_on_streams(gpu_ctx):
    """Captured, replayed with eager calls of another size between, and on two streams at once: the same bits."""
    g = torch.Generator().manual_seed(8)
    mk = lambda rows, vocab, width: dict(  # noqa: E731
        z=torch.randn((rows, vocab), generator=g).cuda(), s=torch.zeros(rows).cuda(), o=torch.zeros(rows).cuda(),
        p=torch.zeros(rows, dtype=I32).cuda(), t=torch.zeros(rows, dtype=I32).cuda(), w=width,
        h=torch.arange(rows * 900, dtype=I32).view(rows, 900).cuda(), ho=torch.zeros((rows, 900), dtype=I32).cuda())
    a, b = mk(60, 8194, 3), mk(32, 50000, 4)

    def call(x, stream=None):
        gpu_ctx.beam_step(x["z"], x["w"], x["s"], x["o"], x["p"], x["t"], states=[(x["h"], x["ho"])], stream=stream)

    def result(x):
        return [x[n].clone() for n in ("o", "p", "t", "ho")]

    call(a), call(b)
    want_b = result(b)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(a)
    for step in range(4):
        a["z"].normal_()
        call(a)
        want = result(a)
        a["o"].zero_(), a["ho"].zero_()
        graph.replay()
        call(b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(result(a), want)) and all(torch.equal(x, y) for x, y in zip(result(b), want_b))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        call(a, streams[0]), call(b, streams[1])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(result(a), want)) and all(torch.equal(x, y) for x, y in zip(result(b), want_b))


def test_nothing_and_refusals(gpu_ctx):
    z = lambda *s, t=F32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    ok = dict(logits=z(6, 40), width=3, score=z(6), out_score=z(6), parent=z(6, t=I32), token=z(6, t=I32))
    gpu_ctx.beam_step(**{**ok, "logits": z(0, 40), "score": z(0), "out_score": z(0), "parent": z(0, t=I32), "token": z(0, t=I32)})
    bits = z(6, 2, t=I32)
    for kw, what in ((dict(stop_token=40), "stop_token"), (dict(stop_token=-2), "stop_token"), (dict(done=z(6, t=U8)), "stop token"),
                     (dict(pen=z(6)), "hist_bits")):
        with pytest.raises(c4s.C4SError, match=f"code 1.*{what}"):
            gpu_ctx.beam_step(**ok, **kw)
    with pytest.raises(c4s.C4SError, match="code 1.*width"):
        wide = {n: (x.repeat(11, *[1] * (x.dim() - 1)) if torch.is_tensor(x) else 33) for n, x in ok.items()}
        gpu_ctx.beam_step(**wide)
    with pytest.raises(c4s.C4SError, match="code 1.*vocab"):
        gpu_ctx.beam_step(**{**ok, "logits": z(6, 0)})
    for kw in (dict(width=4), dict(width=0), dict(score=z(5)), dict(out_score=z(6, t=torch.float64)), dict(parent=z(6)), dict(done=z(6)),
               dict(logits=z(6, 40, t=torch.float16)), dict(hist_bits=z(6, 3, t=I32)), dict(states=[(z(6, 3), z(6, 4))]),
               dict(states=[(z(5, 3), z(5, 3))]), dict(states=[(bits, bits)] * 9), dict(states=[(z(6, 3, t=U8), z(6, 3, t=U8))]),
               dict(temp=z(3))):
        with pytest.raises(ValueError):
            gpu_ctx.beam_step(**{**ok, **kw})
    assert math.isfinite(ok["out_score"].sum().item())
    torch.cuda.synchronize()
