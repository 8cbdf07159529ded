"""The C ABI of the batch's operators without a GPU: exports, struct layouts, null contexts, host tensors, and the
CPU references that the GPU tests use, against each other's definitions."""
import ctypes as C
import subprocess

import numpy as np
import pytest
import torch

import batch_util as B
import c4s

I32, BF, F32, F64 = torch.int32, torch.bfloat16, torch.float32, torch.float64


def test_exports_every_symbol():
    names = c4s.header_functions(c4s.BATCH_HEADER)
    assert sorted(names) == ["c4s_beam_step", "c4s_kv_copy", "c4s_pages_fork", "c4s_pages_grow", "c4s_pages_trim", "c4s_rope"]
    for n in names:
        assert hasattr(c4s.lib(), n)


def test_null_context_is_einval():
    L = c4s.lib()
    assert L.c4s_rope(None, None, None) == c4s.EINVAL
    assert L.c4s_pages_grow(None, None, None, None) == c4s.EINVAL
    assert L.c4s_pages_trim(None, None, None, None) == c4s.EINVAL
    assert L.c4s_pages_fork(None, None, None, 1, None) == c4s.EINVAL
    assert L.c4s_kv_copy(None, None, None, 0, None) == c4s.EINVAL
    assert L.c4s_beam_step(None, None, None) == c4s.EINVAL


def test_ctypes_structs_match_the_header(tmp_path):
    structs = {"c4s_rope_desc": c4s.Rope, "c4s_pages": c4s.PagesDesc, "c4s_grow": c4s.Grow, "c4s_beam_state": c4s.BeamState,
               "c4s_beam": c4s.Beam}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{c4s.BATCH_HEADER}"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'  printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    lines += ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            cname, what, val = line.split()
            py = structs[cname]
            assert int(val) == (C.sizeof(py) if what == "size" else getattr(py, what).offset), line


class _Unreachable:
    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was reached")
        return call


@pytest.fixture
def ctx(monkeypatch):
    """A context of device 0, which no tensor of these tests is on."""
    c4s._Torch.load()
    monkeypatch.setattr(c4s, "_lib", _Unreachable())
    c = object.__new__(c4s.Context)
    c._h, c.device = c4s._vp(), 0
    return c


def test_calls_refuse_host_tensors(ctx):
    z = lambda *s, t=BF: torch.zeros(s, dtype=t)  # noqa: E731
    pages = type("P", (), dict(n_seqs=2, device=0, packed=b""))
    elsewhere = type("P", (), dict(n_seqs=2, device=-1, packed=b""))
    cache = type("C", (), dict(device=0, packed=b""))
    n = z(2, t=I32)
    for call in (lambda: ctx.rope(z(2, 2, 64), None, z(32, t=F64), pos=n),
                 lambda: ctx.pages_grow(elsewhere),
                 lambda: ctx.pages_grow(pages, n),
                 lambda: ctx.pages_trim(pages, n),
                 lambda: ctx.pages_fork(pages, n, 2),
                 lambda: ctx.kv_copy(cache, z(2, 2, t=I32)),
                 lambda: ctx.beam_step(z(2, 10), 2, z(2, t=F32), z(2, t=F32), n, n)):
        with pytest.raises(ValueError, match="cuda:0"):
            call()


def test_pages_of_host_tensors_are_refused():
    z = lambda *s: torch.zeros(s, dtype=I32)  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        c4s.Pages(z(2, 3), z(2), z(6), z(1), 16)


@pytest.mark.parametrize("by", ["none", "linear", "base", "parts"])
def test_rope_freqs(by):
    f = c4s.rope_freqs(64, 10000.0, 4.0, by, trained=2048, device="cpu")
    i = torch.arange(32, dtype=F64)
    plain = 10000.0 ** (-2 * i / 64)
    assert f.dtype == F64 and f.shape == (32,)
    if by == "none":
        assert torch.equal(f, plain)
    elif by == "linear":
        assert torch.equal(f, plain / 4)
    elif by == "base":   # the fastest as it was, the slowest a fourth
        assert f[0] == 1 and abs(f[-1] * 4 / plain[-1] - 1) < 1e-12 and (f[1:] < plain[1:]).all()
    else:
        turns = 2048 * plain / (2 * np.pi)
        assert torch.equal(f[turns > 4], plain[turns > 4]) and torch.equal(f[turns < 1], plain[turns < 1] / 4)
        mid = (turns > 1) & (turns < 4)
        assert mid.any() and (f[mid] < plain[mid]).all() and (f[mid] > plain[mid] / 4).all()
    for bad in (lambda: c4s.rope_freqs(63), lambda: c4s.rope_freqs(64, by="some"), lambda: c4s.rope_freqs(64, by="parts")):
        with pytest.raises(ValueError):
            bad()


def test_quantise4_by_hand():
    x = torch.zeros(32, dtype=BF)
    x[:9] = torch.tensor([6.0, -5.0, 3.5, 2.5, 0.25, 0.75, -0.3, 1.25, 1.75])
    code, e = B.quantise4(x)
    assert e.tolist() == [127]
    # 5 lies halfway between 4 (code 6) and 6 (code 7), 3.5 between 5 and 6, 2.5 between 4 and 5, and so on
    assert code[:9].tolist() == [7, 14, 6, 4, 0, 2, 9, 2, 4]
    assert B.values4(code, e)[:9].tolist() == [6.0, -4.0, 4.0, 2.0, 0.0, 1.0, -0.5, 1.0, 2.0]
    x[0] = 6.03125
    assert B.quantise4(x)[1].tolist() == [128]
    x[0] = float("inf")
    assert B.quantise4(x)[1].tolist() == [255]
    assert B.quantise4(torch.zeros(32, dtype=BF))[1].tolist() == [0]


def test_the_pool_by_hand():
    p = B.Pool(4, 3, 6, 16)
    off, pos, slot, _ = p.grow([17, 0, 16, 0])
    assert p.table == [[0, 1, -1], [-1] * 3, [2, -1, -1], [-1] * 3] and off == [0, 17, 17, 33, 33]
    assert pos[16] == 16 and slot[16] == 16 and slot[17] == 32
    p.fork([0, 0, 0, 0], 2)
    assert p.refs == [2, 2, 2, 0, 0, 0] and p.lens == [17, 17, 16, 16]
    _, _, _, pairs = p.grow(None, True)
    # sequence 0 leaves page 1 to sequence 1; 2 and 3 begin new pages, and one is missing
    assert pairs == [(1, 3), (-1, -1), (-1, -1), (-1, -1)]
    assert p.table == [[0, 3, -1], [0, 1, -1], [2, 4, -1], [2, 5, -1]] and p.missing == 0
    p.trim([18, 2, 1, 1])
    assert p.refs == [1, 0, 2, 0, 0, 0] and p.lens == [0, 16, 16, 16]


def test_beams_by_hand():
    z = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.6, 0.3]], np.float32))
    parent, token, total, done, _ = B.beams(z, 2, np.array([0, -np.inf], np.float32), None, 1)
    assert parent.tolist() == [0, 0] and token.tolist() == [0, 1] and done.tolist() == [False, True]
    parent, token, total, done, _ = B.beams(z, 2, np.log(np.array([0.4, 0.3], np.float32)), [0, 1], 2)
    assert parent.tolist() == [1, 0] and token.tolist() == [2, 0] and done.tolist() == [True, False]
    assert np.allclose(np.exp(total), [0.3, 0.2], rtol=1e-6)
