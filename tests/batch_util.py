"""The batch's operators (include/c4s_batch.h) and the 4-bit cache on the CPU: literal
loops and float64, with nothing of the kernels' ways."""
import math

import numpy as np
import torch

import layers_util as L

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---- 4-bit rows -----------------------------------------------------------------------

def quantise4(x):
    """(codes uint8 [..., dim], exponents + 127 uint8 [..., dim / 32]) of rows of the last dimension."""
    block = x.double().unflatten(-1, (-1, 32))
    top = block.abs().amax(-1)
    fine = torch.isfinite(top)
    e = torch.full(top.shape, -127, dtype=torch.int64)
    for k in range(126, -128, -1):   # the smallest power of two with which nothing exceeds 6
        e = torch.where(fine & (top <= 6 * 2.0 ** k), k, e)
    a = block.abs() / torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())[..., None]
    code, best = torch.zeros_like(a, dtype=torch.int64), torch.full_like(a, math.inf)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):   # the nearest, halfway the even one
        far = (a - GRID[c]).abs()
        code, best = torch.where(far < best, c, code), torch.minimum(far, best)
    code = code + 8 * torch.signbit(block).long()
    return code.flatten(-2).to(torch.uint8), torch.where(fine, e + 127, 255).to(torch.uint8)


def values4(code, e):
    """float64 [..., dim] of codes [..., dim] and bytes [..., dim / 32]; a byte of 255 is NaN, and 4 * 2^126, which is
    past bf16's (and float32's) largest value, infinite."""
    grid = torch.tensor(GRID + [-g for g in GRID], dtype=torch.float64)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double() - 127)
    scale = torch.where(e == 255, math.nan, scale)
    x = grid[code.long()] * scale.repeat_interleave(32, -1)
    return torch.where(x.abs() >= 2.0 ** 128, torch.sign(x) * math.inf, x)


class Cache4(L.Cache):
    """layers_util.Cache in 4 bits. junk: whether unused places hold blocks that are not finite."""

    def __init__(self, lens, heads, dim, page, seed, spare=2, junk=False):
        super().__init__(lens, heads, dim, page, False, seed, spare)
        self.q8 = False
        used = torch.zeros(self.n_pages, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for p in range(n):
                used[self.table[b, p // page], p % page] = True
        g = torch.Generator().manual_seed(seed + 1)
        for name in "kv":
            x = L.bf16((self.n_pages, heads, page, dim), g)
            x = (x.float() * torch.exp(0.7 * torch.randn((heads, 1, dim), generator=g))).to(torch.bfloat16)
            code, e = quantise4(x)
            if junk:
                e = torch.where(used[:, None, :, None], e, torch.tensor(255, dtype=torch.uint8))
            byte = code[..., 0::2] | code[..., 1::2] << 4
            self.t[name] = byte.contiguous() if name == "k" else byte.transpose(2, 3).contiguous()
            self.t[name + "_scale"] = e.transpose(2, 3).contiguous()

    def _of(self, name, pg, at):
        """Rows [n][heads][dim] at places of pages."""
        byte = self.t[name][pg, :, at] if name == "k" else self.t[name][pg, :, :, at]
        code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
        return values4(code, self.t[name + "_scale"][pg, :, :, at])

    def rows(self, name, b, n):
        pos = torch.arange(n)
        i = pos // self.page
        pg = torch.where(i < self.table.shape[1], self.table[b, i.clamp(max=self.table.shape[1] - 1)].long(), torch.tensor(-1))
        there = (pg >= 0) & (pg < self.n_pages)
        return self._of(name, torch.where(there, pg, torch.tensor(0)), pos % self.page), there

    def row(self, name, b, pos):
        i = pos // self.page
        if i >= self.table.shape[1] or not 0 <= int(self.table[b, i]) < self.n_pages:
            return None
        return self._of(name, torch.tensor([int(self.table[b, i])]), torch.tensor([pos % self.page]))[0]

    def spoil(self, name, b, pos, head=None, block=None):
        """A block (all of them) of a position is not finite."""
        pg, at = int(self.table[b, pos // self.page]), pos % self.page
        self.t[name + "_scale"][pg, slice(None) if head is None else head, slice(None) if block is None else block, at] = 255


# ---- rotary positions ---------------------------------------------------------------------

def rope(x, pos, freq, pairs, scale):
    """(result, size of what it is made of) of rows [rows][heads][dim] in float64; rows at positions below 0 as they are."""
    y, rot = L.f64(x).clone(), 2 * len(freq)
    angle = pos.double()[:, None] * freq.cpu().double()
    cos, sin = (f(angle)[:, None] * scale for f in (torch.cos, torch.sin))
    at = torch.arange(rot).view(-1, 2).t() if pairs else torch.arange(rot).view(2, -1)
    a, b = y[..., at[0]], y[..., at[1]]
    size = torch.zeros_like(y)
    y[..., at[0]], y[..., at[1]] = a * cos - b * sin, a * sin + b * cos
    size[..., at[0]] = size[..., at[1]] = (a.abs() + b.abs()) * abs(scale)
    y[pos < 0], size[pos < 0] = L.f64(x)[pos < 0], 0
    return y, size


# ---- pages ------------------------------------------------------------------------------------

class Pool:
    """Tables, counts and free pages as plain lists, a sequence at a time."""

    def __init__(self, n_seqs, max_pages, n_pages, page):
        self.n, self.max_pages, self.n_pages, self.page = n_seqs, max_pages, n_pages, page
        self.lens, self.refs, self.missing = [0] * n_seqs, [0] * n_pages, 0
        self.table = [[-1] * max_pages for _ in range(n_seqs)]

    def device(self):
        import c4s
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
        return c4s.Pages(i32(self.table).view(self.n, self.max_pages), i32(self.lens), i32(self.refs), i32(self.free_words()),
                         self.page, i32([self.missing]))

    def free_words(self):
        words = np.zeros((self.n_pages + 31) // 32, np.uint32)
        for p, r in enumerate(self.refs):
            if r == 0:
                words[p // 32] |= np.uint32(1 << p % 32)
        return words.view(np.int32).tolist()

    def same(self, pages):
        assert pages.lens.tolist() == self.lens
        assert pages.block_table.tolist() == self.table
        assert pages.refs.tolist() == self.refs
        assert pages.free_bits.tolist() == self.free_words()
        assert pages.missing.tolist() == [self.missing]

    def _pages(self, tokens):
        return min(-(-tokens // self.page), self.max_pages)

    def grow(self, new=None, copies=False):
        """(rows_off, positions, slots, copies)."""
        new = [1] * self.n if new is None else [max(x, 0) for x in new]
        pairs = [(-1, -1)] * self.n
        own = [None] * self.n    # the shared last page that a sequence gives up
        if copies:
            holds = {}
            for b in range(self.n):
                at = self.lens[b] // self.page
                if new[b] and self.lens[b] % self.page and at < self.max_pages:
                    p = self.table[b][at]
                    if 0 <= p < self.n_pages and self.refs[p] > 1:
                        holds.setdefault(p, []).append(b)
            for p, users in holds.items():
                for b in users[:-1] if len(users) == self.refs[p] else users:
                    own[b] = p
            for p in own:
                if p is not None:
                    self.refs[p] -= 1
        free = [p for p in range(self.n_pages) if self.refs[p] == 0]   # a page given up is still held by somebody
        for b in range(self.n):
            have, want = self._pages(self.lens[b]), self._pages(self.lens[b] + new[b])
            at = ([self.lens[b] // self.page] if own[b] is not None else []) + list(range(have, want))
            for nth, i in enumerate(at):
                p = free.pop(0) if free else -1
                self.table[b][i] = p
                if p >= 0:
                    self.refs[p] = 1
                    if own[b] is not None and nth == 0:
                        pairs[b] = (own[b], p)
                else:
                    self.missing += 1
            tokens = self.lens[b] + new[b]
            self.missing += (-(-tokens // self.page) - want) - (-(-self.lens[b] // self.page) - have)
        off, pos, slot = [0], [], []
        for b in range(self.n):
            for t in range(self.lens[b], self.lens[b] + new[b]):
                i = t // self.page
                p = self.table[b][i] if i < self.max_pages else -1
                pos.append(t)
                slot.append(p * self.page + t % self.page if 0 <= p < self.n_pages else -1)
            self.lens[b] += new[b]
            off.append(off[-1] + new[b])
        return off, pos, slot, pairs

    def trim(self, drop):
        for b in range(self.n):
            left = max(self.lens[b] - max(drop[b], 0), 0)
            for i in range(self._pages(left), self._pages(self.lens[b])):
                if 0 <= self.table[b][i] < self.n_pages:
                    self.refs[self.table[b][i]] -= 1
                self.table[b][i] = -1
            self.lens[b] = left

    def fork(self, parent, width):
        table, lens = [list(r) for r in self.table], list(self.lens)
        for b in range(self.n):
            for p in table[b]:
                if 0 <= p < self.n_pages:
                    self.refs[p] -= 1
        for b in range(self.n):
            ok = 0 <= parent[b] < width
            src = b // width * width + parent[b]
            self.table[b] = list(table[src]) if ok else [-1] * self.max_pages
            self.lens[b] = lens[src] if ok else 0
            for p in self.table[b]:
                if 0 <= p < self.n_pages:
                    self.refs[p] += 1


# ---- beams ----------------------------------------------------------------------------------------

def beams(logits, width, score, done=None, stop=-1, temp=None, pen=None, bits=None):
    """(parent, token, total float64, done, bits) of every row, by a sort of all candidates in float64. logits, score,
    temp, pen: float32 arrays; bits: bool [rows][vocab]."""
    z = np.array(logits, np.float32)
    rows, vocab = z.shape
    out = [np.zeros(rows, np.int64), np.zeros(rows, np.int64), np.zeros(rows), np.zeros(rows, bool),
           None if bits is None else np.zeros_like(bits)]
    for r in range(rows):
        with np.errstate(invalid="ignore"):
            if pen is not None and pen[r] != 1:
                hit = bits[r]
                z[r] = np.where(hit, np.where(z[r] < 0, z[r] * pen[r], z[r] / pen[r]), z[r])
            if temp is not None and temp[r] > 0 and temp[r] != 1:
                z[r] = z[r] / temp[r]
    for g in range(rows // width):
        total = np.full((width, vocab), -np.inf)
        offered = np.ones((width, vocab), bool)
        for j in range(width):
            r = g * width + j
            if done is not None and done[r]:
                offered[j] = False
                offered[j, stop], total[j, stop] = True, score[r]
            elif score[r] > -np.inf and z[r].max() > -np.inf:
                x = z[r].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    t = np.float64(score[r]) + ((x - x.max()) - np.log(np.exp(x - x.max()).sum()))   # (the log counts beside 1e38 too)
                total[j] = np.where(np.isnan(t), -np.inf, t)
        at = np.flatnonzero(offered)
        best = at[np.argsort(-total.reshape(-1)[at], kind="stable")[:width]]
        for i, c in enumerate(best):
            r, j, v = g * width + i, c // vocab, c % vocab
            src = g * width + j
            was = bool(done is not None and done[src])
            out[0][r], out[1][r], out[2][r], out[3][r] = j, v, total[j, v], was or v == stop
            if bits is not None:
                out[4][r] = bits[src]
                if not out[3][r]:
                    out[4][r, v] = True
    return out


def pack_bits(bits):
    """bool [rows][vocab] as int32 words."""
    rows, vocab = bits.shape
    full = np.zeros((rows, (vocab + 31) // 32 * 32), np.uint8)
    full[:, :vocab] = bits
    return torch.from_numpy(np.packbits(full, axis=1, bitorder="little").view(np.int32).copy())
