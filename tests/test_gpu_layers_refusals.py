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
