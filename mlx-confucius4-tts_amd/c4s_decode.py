"""A pre-norm decoder in front of the token-sampling step, from the decoder
layer's operators (include/c4s_layers.h): prompts, then one token a sequence and
step, every step one graph replay from the last tokens to the next.

    python mlx-confucius4-tts_amd/c4s_decode.py --rows 64 --layers 4 --tokens 100

runs it with random weights and prints the time of a step. The layer's order is
that of the reference's GPT-2 (src/t2s/gpt2.cpp): norm, attention, residual,
norm, MLP, residual, with the final norm inside the LM head.
"""
from __future__ import annotations

import argparse

import torch

import c4s

ACT = "gelu"


def random_weights(layers: int, dim: int, heads: int, kv_heads: int, vocab: int, positions: int, seed: int = 0,
                   device="cuda") -> dict:
    """Weights as Decoder takes them; projections stored (out, in)."""
    g = torch.Generator().manual_seed(seed)
    hd = dim // heads

    def w(*shape, std=0.02, dtype=torch.bfloat16, mean=0.0):
        return (torch.randn(shape, generator=g) * std + mean).to(dtype).to(device)

    f = torch.float32
    layer = lambda: dict(norm1=(w(dim, dtype=f, mean=1.0), w(dim, dtype=f)), norm2=(w(dim, dtype=f, mean=1.0), w(dim, dtype=f)),  # noqa: E731
                         qkv=w((heads + 2 * kv_heads) * hd, dim), qkv_bias=w((heads + 2 * kv_heads) * hd, dtype=f),
                         out=w(dim, dim), out_bias=w(dim, dtype=f), up=w(4 * dim, dim), up_bias=w(4 * dim, dtype=f),
                         down=w(dim, 4 * dim), down_bias=w(dim, dtype=f))
    return dict(layers=[layer() for _ in range(layers)], tokens=w(vocab, dim), positions=w(positions, dim),
                final_norm=(w(dim, dtype=f, mean=1.0), w(dim, dtype=f)), head=w(vocab, dim), head_bias=w(vocab, dtype=f))


class Decoder:
    """One batch of sequences: begin(prompts), then step() for each further token.

    Sequences get their pages from one pool of `n_pages` when the batch begins,
    for as many tokens as it may come to hold: `room` further steps are left."""

    def __init__(self, ctx: c4s.Context, weights: dict, heads: int, kv_heads: int, n_pages: int, page_size: int = 16,
                 q8_cache: bool = False):
        self.ctx, self.w, self.heads, self.kv_heads = ctx, weights, heads, kv_heads
        self.vocab, self.dim = weights["tokens"].shape
        self.hd, self.page_size, self.n_pages = self.dim // heads, page_size, n_pages
        table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
        self.caches = [c4s.KvCache.empty(n_pages, kv_heads, page_size, self.hd, table, q8=q8_cache)
                       for _ in weights["layers"]]
        self.room = 0

    def _buffers(self, rows: int) -> dict:
        e = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        return dict(x=torch.empty((rows, self.dim), device="cuda"), h=e(rows, self.dim), a=e(rows, self.heads, self.hd),
                    qkv=e(rows, self.heads + 2 * self.kv_heads, self.hd), m=e(rows, 4 * self.dim))

    def _layers(self, b: dict, rows_off, max_new: int) -> None:
        """The residual stream b["x"] through every layer; the new tokens' keys and values join the caches."""
        ctx, rows, H, K = self.ctx, b["x"].shape[0], self.heads, self.kv_heads
        for w, cache in zip(self.w["layers"], self.caches):
            ctx.block_norm(b["x"], *w["norm1"], b["h"])
            ctx.linear(b["h"], w["qkv"], b["qkv"].view(rows, -1), bias=w["qkv_bias"])
            ctx.kv_append(cache, b["qkv"][:, H:H + K], b["qkv"][:, H + K:], self.lens, rows_off)
            ctx.attn(b["qkv"][:, :H], cache, self.lens, b["a"], rows_off=rows_off, max_new=max_new)
            ctx.linear(b["a"].view(rows, -1), w["out"], b["x"], bias=w["out_bias"], residual=b["x"])
            ctx.block_norm(b["x"], *w["norm2"], b["h"])
            ctx.linear(b["h"], w["up"], b["m"], bias=w["up_bias"], act=ACT)
            ctx.linear(b["m"], w["down"], b["x"], bias=w["down_bias"], residual=b["x"])

    def begin(self, prompts: list, max_new: int) -> torch.Tensor:
        """Prompts (lists of ids) into the caches, with room for max_new further tokens each; the last hidden row of
        each, bf16 [sequences][dim]."""
        self.room = 0
        n = [len(p) for p in prompts]
        if not n or max_new < 0:
            raise ValueError("no prompts, or max_new below 0")
        need = [-(-(k + max_new) // self.page_size) for k in n]
        if min(n) < 1 or sum(need) > self.n_pages or max(n) + max_new > self.w["positions"].shape[0]:
            raise ValueError("empty prompt, or more tokens than pages or positions")
        ids = torch.cat([torch.as_tensor(p) for p in prompts])
        if int(ids.min()) < 0 or int(ids.max()) >= self.vocab:   # on the device an index out of range ends the process
            raise ValueError("a prompt's id is outside the vocabulary")
        table = torch.full((len(n), max(need)), -1, dtype=torch.int32)
        at = 0
        for row, k in zip(table, need):
            row[:k] = torch.arange(at, at + k, dtype=torch.int32)
            at += k
        table = table.cuda()
        self.caches = [c4s.KvCache(c.k, c.v, table, c.k_scale, c.v_scale) for c in self.caches]
        self.lens = torch.tensor(n, dtype=torch.int32, device="cuda")
        ids = ids.cuda()
        pos = torch.cat([torch.arange(k) for k in n]).cuda()
        off = torch.zeros(len(n) + 1, dtype=torch.int32)
        off[1:] = torch.tensor(n).cumsum(0)
        b = self._buffers(len(ids))
        torch.add(self.w["tokens"][ids].float(), self.w["positions"][pos].float(), out=b["x"])
        self._layers(b, off.cuda(), max(n))
        self.one = self._buffers(len(n))   # a step's
        self.room = max_new
        return b["x"][(off[1:] - 1).cuda().long()].bfloat16()

    def step(self, tokens) -> torch.Tensor:
        """One more token a sequence (int32 or int64 [sequences], ids of the vocabulary); its hidden row, bf16. May be
        captured into a graph, whose replays are the caller's to count."""
        if self.room < 1:
            raise ValueError("no room for a further token: begin() gives as many steps as its max_new")
        self.room -= 1
        b = self.one
        torch.add(self.w["tokens"][tokens].float(), self.w["positions"][self.lens].float(), out=b["x"])
        self.lens.add_(1)
        self._layers(b, None, 1)
        return b["x"].bfloat16()

    def generate(self, prompts: list, max_new: int, temp, top_k, top_p, pen, rng, graph: bool = True) -> torch.Tensor:
        """max_new sampled tokens of each prompt, int32 [sequences][max_new]; rng (int64 [sequences]) is advanced.
        temp, top_k, top_p, pen: one value a sequence, on the device. graph: steps as replays of one graph."""
        if max_new < 1:
            raise ValueError("max_new below 1")
        R, w = len(prompts), self.w
        bits = torch.zeros((R, (self.vocab + 31) // 32), dtype=torch.int32, device="cuda")
        token = torch.empty(R, dtype=torch.int32, device="cuda")
        out = torch.empty((R, max_new), dtype=torch.int32, device="cuda")

        def sample(hidden):
            self.ctx.lmhead_sample(hidden, *w["final_norm"], w["head"], w["head_bias"], None, None, temp, top_k, top_p,
                                   pen, rng, token, hist_bits=bits)

        def again():
            sample(self.step(token))

        sample(self.begin(prompts, max_new))
        out[:, 0] = token
        replay = again
        for i in range(1, max_new):
            if graph and i == 2:   # the first step, made eagerly, has sized every workspace
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    again()
                replay = g.replay
            replay()
            out[:, i] = token
        torch.cuda.synchronize()
        return out


def main() -> None:
    p = argparse.ArgumentParser()
    p.add_argument("--rows", type=int, default=64)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--dim", type=int, default=1280)
    p.add_argument("--heads", type=int, default=20)
    p.add_argument("--kv-heads", type=int, default=20)
    p.add_argument("--vocab", type=int, default=8194)
    p.add_argument("--prompt", type=int, default=200)
    p.add_argument("--tokens", type=int, default=100)
    p.add_argument("--q8-cache", action="store_true")
    a = p.parse_args()
    ctx = c4s.Context(0)
    weights = random_weights(a.layers, a.dim, a.heads, a.kv_heads, a.vocab, a.prompt + a.tokens)
    d = Decoder(ctx, weights, a.heads, a.kv_heads, a.rows * (-(-(a.prompt + a.tokens) // 16)), q8_cache=a.q8_cache)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, a.vocab, (a.prompt,), generator=g) for _ in range(a.rows)]
    full = lambda v, t: torch.full((a.rows,), v, dtype=t, device="cuda")  # noqa: E731
    par = (full(0.8, torch.float32), full(30, torch.int32), full(0.8, torch.float32), full(10.0, torch.float32))
    rng = lambda: torch.arange(1, a.rows + 1, device="cuda") * 0x100000001B3  # noqa: E731
    d.generate(prompts, 4, *par, rng())
    t = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
    t[0].record()
    d.generate(prompts, 3, *par, rng())
    t[1].record()
    d.generate(prompts, a.tokens, *par, rng())
    t[2].record()
    torch.cuda.synchronize()
    few, many = t[0].elapsed_time(t[1]), t[1].elapsed_time(t[2])
    print(f"{a.rows} sequences of {a.prompt} tokens, {a.layers} layers of {a.dim}: prompts and three tokens {few:.2f} ms, "
          f"a further step {(many - few) / (a.tokens - 3):.3f} ms")
    ctx.close()


if __name__ == "__main__":
    main()
