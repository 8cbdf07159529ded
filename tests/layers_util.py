"""The decoder layer's operators (include/c4s_layers.h) in float64, on the CPU,
with the bounds that the tests hold the kernels to."""
import numpy as np
import torch

U = 2.0 ** -24    # a float32 rounding
BF16 = 2.0 ** -8  # one bf16 unit: half of it for the rounding, and a whole one where a sum's error crosses a boundary


def f64(t):
    return t.detach().cpu().to(torch.float64)


def bf16(shape, gen, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen) * scale + shift).to(torch.bfloat16)


def norm(v, rms, eps, gamma, beta):
    if not rms:
        v = v - v.mean(-1, keepdim=True)
    v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    if gamma is not None:
        v = v * f64(gamma)
    return v if beta is None else v + f64(beta)


def gelu(y):
    return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))


ACT = {"none": lambda y: y, "gelu": gelu, "silu": lambda y: y * torch.sigmoid(y), "relu": lambda y: y.clamp_min(0)}


def weights64(w, quant):
    """(w, |parts of w|): the weights in float64, and the sum of magnitudes they are computed from."""
    if quant is None:
        return f64(w), f64(w).abs()
    scale, off, group = (f64(quant[0]), f64(quant[1]), quant[2])
    s, b = scale.repeat_interleave(group, 1), off.repeat_interleave(group, 1)
    q = f64(w)
    return q * s + b, ((q - 128) * s).abs() + (b + 128 * s).abs()


def linear(x, w, quant, bias, act, residual):
    """(result, bound on a float32 evaluation's error): K products summed in float32 in any
    order with at most K / 8 + 64 roundings on the way of one of them; the activations' slopes stay below 1.2."""
    w64, mag = weights64(w, quant)
    x64 = f64(x)
    y = x64 @ w64.t()
    err = (x.shape[1] / 8 + 64) * 2 * U * (x64.abs() @ mag.t())
    if bias is not None:
        y = y + f64(bias)
        err = err + U * y.abs()
    y = ACT[act](y)
    err = 1.2 * err + 8 * U * y.abs()
    if residual is not None:
        y = y + f64(residual)
        err = err + U * y.abs()
    return y, err


class Cache:
    """A paged cache on the CPU, filled at random: pages of every sequence in no order,
    `spare` pages that none has, unused places filled with `junk`."""

    def __init__(self, lens, heads, dim, page, q8, seed, spare=2, junk=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lens, self.heads, self.dim, self.page, self.q8 = list(lens), heads, dim, page, q8
        used = torch.zeros(self.n_pages, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for p in range(n):
                used[self.table[b, p // page], p % page] = True
        self.t = {}
        for name in "kv":
            x = bf16((self.n_pages, heads, page, dim), g)
            if q8:
                x, s = quantise(x)
                if junk is not None:
                    s = torch.where(used[:, None, :], s, torch.tensor(junk, dtype=torch.float32))
                self.t[name + "_scale"] = s
            elif junk is not None:
                x = torch.where(used[:, None, :, None], x, torch.tensor(junk, dtype=torch.bfloat16))
            self.t[name] = x.contiguous() if name == "k" else x.transpose(2, 3).contiguous()

    def cuda(self):
        import c4s
        d = {k: v.cuda() for k, v in self.t.items()}
        return c4s.KvCache(d["k"], d["v"], self.table.cuda(), d.get("k_scale"), d.get("v_scale"))

    def update_from(self, kc):
        """The contents of a device cache of this shape."""
        for name in self.t:
            self.t[name] = getattr(kc, name).cpu()

    def row(self, name, b, pos):
        """(value [heads][dim] in float64 or None where there is no page)."""
        i = pos // self.page
        if i >= self.table.shape[1] or not 0 <= int(self.table[b, i]) < self.n_pages:
            return None
        pg, at = int(self.table[b, i]), pos % self.page
        x = self.t[name][pg, :, at] if name == "k" else self.t[name][pg, :, :, at]
        x = x.to(torch.float64)
        return x * self.t[name + "_scale"][pg, :, at, None].to(torch.float64) if self.q8 else x

    def rows(self, name, b, n):
        """(values [n][heads][dim] of sequence b's first n positions in float64, which of them have a page [n])."""
        pos = torch.arange(n)
        i = pos // self.page
        pg = torch.where(i < self.table.shape[1], self.table[b, i.clamp(max=self.table.shape[1] - 1)].long(), torch.tensor(-1))
        there = (pg >= 0) & (pg < self.n_pages)
        pg, at = torch.where(there, pg, torch.tensor(0)), pos % self.page
        x = self.t[name][pg, :, at] if name == "k" else self.t[name][pg, :, :, at]
        x = x.to(torch.float64)
        if self.q8:
            x = x * self.t[name + "_scale"][pg, :, at, None].to(torch.float64)
        return x, there


def quantise(x):
    """8-bit codes and scales of rows of the last dimension, in the float32 steps of the definition."""
    x = x.float()
    scale = x.abs().amax(-1) / np.float32(127)
    q = torch.round(torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros(()))).clamp(-127, 127)
    return q.to(torch.int8), scale


def attn(cache, q, n_new, heads, scale, first=None):
    """(out, lse, sum w|v|, sqrt(sum w^2 v^2)) of packed rows q [rows][heads][dim]; n_new: rows a sequence."""
    rows, dim = q.shape[0], cache.dim
    out, lse = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.full((rows, heads), -np.inf, dtype=torch.float64)
    mag, sq = torch.zeros_like(out), torch.zeros_like(out)
    shared, r = heads // cache.heads, 0
    for b, n in enumerate(n_new):
        length = cache.lens[b]
        keys = [(p, cache.row("k", b, p), cache.row("v", b, p)) for p in range(max(0, first[b]) if first is not None else 0, length)]
        keys = [k for k in keys if k[1] is not None]
        pos = torch.tensor([k[0] for k in keys])
        if keys:
            ks, vs = (torch.stack([k[i] for k in keys]).repeat_interleave(shared, 1) for i in (1, 2))   # [key][head][dim]
        for i in range(n):
            if keys:
                see = pos <= length - n + i
                if see.any():
                    k, v = ks[see], vs[see]
                    z = (k * f64(q[r])[None]).sum(-1) * scale          # [key][head]
                    lse[r] = torch.logsumexp(z, 0)
                    w = torch.exp(z - lse[r])[..., None]
                    out[r] = (w * v).sum(0)
                    mag[r] = (w * v.abs()).sum(0)
                    sq[r] = (w * v).square().sum(0).sqrt()
            r += 1
    return out, lse, mag, sq


def attn_row(cache, b, pos, q, scale, first=0):
    """One row of attn(): q [heads][dim] of sequence b's position pos."""
    heads, shared = q.shape[0], q.shape[0] // cache.heads
    k, there = cache.rows("k", b, pos + 1)
    v, _ = cache.rows("v", b, pos + 1)
    there[:max(0, min(first, pos + 1))] = False
    if not there.any():
        zero = torch.zeros(heads, cache.dim, dtype=torch.float64)
        return zero, torch.full((heads,), -np.inf, dtype=torch.float64), zero, zero
    k, v = (x[there].repeat_interleave(shared, 1) for x in (k, v))
    z = (k * f64(q)[None]).sum(-1) * scale
    lse = torch.logsumexp(z, 0)
    w = torch.exp(z - lse)[..., None]
    return (w * v).sum(0), lse, (w * v.abs()).sum(0), (w * v).square().sum(0).sqrt()
