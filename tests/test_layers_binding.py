"""What the binding of the layer calls refuses before it reaches the library, shown without a GPU: tensors that are
not on the context's device. `_lib` is replaced by one whose calls fail the test."""
import pytest
import torch

import c4s

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


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


def test_helpers_refuse_host_tensors():
    c4s._Torch.load()
    for call in (lambda: c4s._rows(torch.zeros(2, 4), (2, 4), "x", 0),
                 lambda: c4s._heads(torch.zeros(2, 3, 4), (2, 3, 4), "x", 0),
                 lambda: c4s._vector(torch.zeros(4), 4, "x", 0),
                 lambda: c4s._i32(torch.zeros(4, dtype=I32), 4, "x", 0)):
        with pytest.raises(ValueError, match="x.*cuda:0"):
            call()
    # on the device that is asked for (-1: the host's number) they pass
    assert c4s._rows(torch.zeros(2, 4), (2, 4), "x", -1)[1:] == (4, c4s.F32)
    assert c4s._vector(None, 4, "x", 0) == 0 and c4s._i32(None, 4, "x", 0) == 0


def test_a_cache_of_host_tensors_is_refused():
    k, v, table = torch.zeros(3, 2, 16, 64, dtype=BF), torch.zeros(3, 2, 64, 16, dtype=BF), torch.zeros(1, 3, dtype=I32)
    with pytest.raises(ValueError, match="GPU"):
        c4s.KvCache(k, v, table)
    q, s = torch.int8, torch.zeros(3, 2, 16)
    with pytest.raises(ValueError, match="GPU"):
        c4s.KvCache(k.to(q), v.to(q), table, s, s)


def test_calls_refuse_host_tensors(ctx):
    z = lambda *s, t=BF: torch.zeros(s, dtype=t)  # noqa: E731
    cache = type("C", (), dict(n_kv_heads=2, head_dim=64, n_seqs=2, device=0, packed=b""))
    lens = z(2, t=I32)
    for call in (lambda: ctx.block_norm(z(2, 8), None, None, z(2, 8)),
                 lambda: ctx.linear(z(2, 64), z(4, 64), z(2, 4)),
                 lambda: ctx.kv_append(cache, z(2, 2, 64), z(2, 2, 64), lens),
                 lambda: ctx.kv_read(cache, z(2, 2, 64), z(2, 2, 64), lens),
                 lambda: ctx.attn(z(2, 2, 64), cache, lens, z(2, 2, 64))):
        with pytest.raises(ValueError, match="cuda:0"):
            call()
