"""What the layer calls refuse, argument by argument. Nothing here is queued."""
import pytest
import torch

import c4s

pytestmark = pytest.mark.gpu

BF, F32, I32, U8, I8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8, torch.int8


def z(*s, t=BF):
    return torch.zeros(s, dtype=t, device="cuda")


def _each_on_the_host(call, args, match):
    """call(**args) works; with any one tensor of args in host memory it does not."""
    call(**args)
    for name, t in args.items():
        if isinstance(t, torch.Tensor):
            print(f"{name} on the host", flush=True)
            with pytest.raises(ValueError, match=match):
                call(**{**args, name: t.cpu()})
    torch.cuda.synchronize()


def test_host_tensors(gpu_ctx):
    v = lambda n: z(n, t=F32)  # noqa: E731
    _each_on_the_host(gpu_ctx.block_norm, dict(
        x=z(4, 8), gamma=v(8), beta=v(8), out=z(4, 8), y=z(4, 8), x_out=z(4, 8), post=True, post_gamma=v(8),
        post_beta=v(8), gate=z(2, 8, t=F32), gate_rows=2), "cuda:0")
    _each_on_the_host(gpu_ctx.linear, dict(x=z(2, 64), weight=z(4, 64), out=z(2, 4), bias=v(4), residual=z(2, 4)), "cuda:0")
    _each_on_the_host(
        lambda x, weight, out, s, o: gpu_ctx.linear(x, weight, out, quant=(s, o, 32)),
        dict(x=z(2, 64), weight=z(4, 64, t=U8), out=z(2, 4), s=z(4, 2, t=F32), o=z(4, 2, t=F32)), "cuda:0")
    kc = c4s.KvCache(z(3, 2, 16, 64), z(3, 2, 64, 16), z(2, 3, t=I32))
    lens, off = torch.tensor([1, 1], dtype=I32).cuda(), torch.tensor([0, 1, 2], dtype=I32).cuda()
    rows = dict(cache=kc, k=z(2, 2, 64), v=z(2, 2, 64), lens=lens, rows_off=off)
    _each_on_the_host(gpu_ctx.kv_append, rows, "cuda:0")
    _each_on_the_host(gpu_ctx.kv_read, rows, "cuda:0")
    _each_on_the_host(gpu_ctx.attn, dict(q=z(2, 2, 64), cache=kc, lens=lens, out=z(2, 2, 64), rows_off=off,
                                         first=z(2, t=I32), lse=z(2, 2, t=F32)), "cuda:0")
    _each_on_the_host(c4s.KvCache, dict(k=z(3, 2, 16, 64, t=I8), v=z(3, 2, 64, 16, t=I8), block_table=z(2, 3, t=I32),
                                        k_scale=z(3, 2, 16, t=F32), v_scale=z(3, 2, 16, t=F32)), "GPU")


@pytest.mark.parametrize("M,N,what", [(2 ** 31 - 1, 4, b"1073741824"), (2 ** 31 - 200, 4, b"1073741824"),
                                      (2 ** 30 + 1, 4, b"1073741824"), (2 ** 30, 129, b"16777208"),
                                      (128 * 32768 + 1, 65536, b"16777208"), (2 ** 23, 2 ** 22, b"16777208")])
def test_linear_past_a_grid(gpu_ctx, M, N, what):
    """Within 255 of 2^31 rows a count of tiles in 32 bits turns negative; from 2^24 tiles on the grid has 2^32
    threads. Nothing is queued: the addresses are of small tensors."""
    x, w, out = z(16, 64), z(16, 64), z(16, 64)
    desc = c4s._pack_linear(M, N, 64, 0, x.data_ptr(), 64, w.data_ptr(), c4s.W_BF16, 0, 0, 0, 0, 0, 0, c4s.F32, c4s.BF16,
                            out.data_ptr(), N)
    assert c4s.lib().c4s_linear(gpu_ctx._h, desc, None) == c4s.EINVAL
    assert what in c4s.lib().c4s_last_error(gpu_ctx._h)
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_linear_of_many_short_rows(gpu_ctx):
    """2^28 + 3 rows of 8 inputs, past 2^32 bytes, and one output each."""
    M = (1 << 28) + 3
    g = torch.Generator().manual_seed(3)
    small = torch.randint(-4, 5, (4099, 8), generator=g).to(BF).cuda()     # exact in every order
    w = torch.randint(-4, 5, (1, 8), generator=g).to(BF).cuda()
    x = small.repeat(-(-M // 4099), 1)[:M]
    out = torch.empty((M, 1), device="cuda")
    gpu_ctx.linear(x, w, out)
    assert torch.equal(out[:, 0], (small.float() * w.float()).sum(1).repeat(-(-M // 4099))[:M])


def test_attn_past_a_grid(gpu_ctx):
    """65535 key heads, three tiles of query heads each, 128 parts of 2^21 positions: 2^32 threads and more. Refused
    before any workspace is made; nothing is queued: the addresses are of small tensors."""
    p, s, i = z(16, 64).data_ptr(), z(16, 64, t=F32).data_ptr(), z(64, t=I32).data_ptr()
    heads, pages, shared = 65535, 131072, 48
    cache = bytes(c4s.KvCacheDesc(p, p, s, s, i, pages, 1, pages, 1, 16, heads, 16, c4s.KV_Q8))
    attn = c4s._pack_attn(p, heads * shared * 16, p, heads * shared * 16, 0, i, 0, 0, 1, 1, heads * shared, 0.25)
    free = torch.cuda.mem_get_info()[0]
    assert c4s.lib().c4s_attn(gpu_ctx._h, cache, attn, None) == c4s.EINVAL
    assert b"too many parts" in c4s.lib().c4s_last_error(gpu_ctx._h)
    assert free - torch.cuda.mem_get_info()[0] < 1 << 30
    torch.cuda.synchronize()
