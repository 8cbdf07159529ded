"""Pages handed out, taken back, shared and copied (c4s_pages_*, c4s_kv_copy) against a literal simulation, exactly."""
import random

import pytest
import torch

import batch_util as B
import c4s

pytestmark = pytest.mark.gpu
I32 = torch.int32


def i32(v):
    return torch.tensor(v, dtype=I32).cuda()


def _grow(ctx, pool, pages, new, copies, maps=True, room=None):
    n = pool.n
    total = n if new is None else sum(max(x, 0) for x in new)
    room = total + 5 if room is None else room
    off = torch.full((n + 1,), -9, dtype=I32, device="cuda") if maps else None
    pos, slot = (torch.full((room,), -9, dtype=I32, device="cuda") for _ in "ps") if maps else (None, None)
    pairs = torch.full((n, 2), -9, dtype=I32, device="cuda") if copies else None
    ctx.pages_grow(pages, None if new is None else i32(new), off, pos, slot, pairs)
    want = pool.grow(new, copies)
    pool.same(pages)
    if maps:
        most = min(total, room)
        assert off.tolist() == want[0] and pos.tolist()[:most] == want[1][:most] and slot.tolist()[:most] == want[2][:most]
        assert (pos[most:] == -9).all() and (slot[most:] == -9).all()
    if copies:
        assert [tuple(p) for p in pairs.tolist()] == want[3]
    return want


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page", [16, 64, 256])
def test_a_run_of_calls(gpu_ctx, page, seed):
    """Growing, trimming and forking at random, pools that run out, tables that are too short."""
    r = random.Random(seed * 1000 + page)
    width = r.choice([1, 2, 3, 4, 8, 32])
    n = width * r.randint(1, 9)
    max_pages = r.randint(2, 12)
    pool = B.Pool(n, max_pages, r.choice([3, 31, 32, 33, 100, 400]), page)
    pages = c4s.Pages.empty(n, max_pages, pool.n_pages, page)
    pool.same(pages)
    print(f"pages page={page} seed={seed} n={n} width={width} max={max_pages} pool={pool.n_pages}", flush=True)
    for step in range(14):
        what = r.choice(["grow", "one", "trim", "fork"]) if step else "grow"
        if what == "grow":
            _grow(gpu_ctx, pool, pages, [r.choice([0, 1, r.randint(0, 3 * page), -2]) for _ in range(n)], True,
                  maps=r.random() < 0.8)
        elif what == "one":
            _grow(gpu_ctx, pool, pages, None, True)
        elif what == "trim":
            drop = [r.choice([0, 0, 1, r.randint(0, 2 * page), 2 ** 31 - 1, -3]) for _ in range(n)]
            gpu_ctx.pages_trim(pages, i32(drop))
            pool.trim(drop)
            pool.same(pages)
        else:
            parent = [r.choice([r.randrange(width), j % width, r.choice([-1, width])]) if r.random() < 0.9 else 0 for j in range(n)]
            gpu_ctx.pages_fork(pages, i32(parent), width)
            pool.fork(parent, width)
            pool.same(pages)


@pytest.mark.parametrize("n,pages_n", [(1, 1), (1, 5000), (4096, 9000), (1025, 140000), (7, 300001)])
def test_sizes(gpu_ctx, n, pages_n):
    """One sequence, more than a workgroup's threads, free pages far behind held ones, more than one round of them."""
    r = random.Random(n)
    pool = B.Pool(n, 9, pages_n, 16)
    if pages_n > 100000:   # most of the front is held by somebody else
        for p in range(pages_n * 9 // 10):
            pool.refs[p] = int(r.random() < 0.999)
    pages = pool.device()
    print(f"pages n={n} pool={pages_n}", flush=True)
    _grow(gpu_ctx, pool, pages, [r.randint(0, 40) for _ in range(n)], False)
    _grow(gpu_ctx, pool, pages, None, True)
    drop = [r.randint(0, 60) for _ in range(n)]
    gpu_ctx.pages_trim(pages, i32(drop))
    pool.trim(drop)
    pool.same(pages)
    _grow(gpu_ctx, pool, pages, [r.randint(0, 90) for _ in range(n)], True, room=3)


def test_rows_of_many_tokens(gpu_ctx):
    """Maps that the one workgroup writes, and maps of their own kernel, at the border between them."""
    for n, new, room in ((3, 2000, None), (64, 32, None), (64, 33, None), (4096, 1, 4096), (200, 10, 2049), (1, 9000, 70)):
        print(f"maps n={n} new={new} room={room}", flush=True)
        pool = B.Pool(n, 700, 12000, 16)
        pages = pool.device()
        for step in range(2):
            _grow(gpu_ctx, pool, pages, [new + (b + step) % 2 for b in range(n)], step == 1, room=room)


def test_more_tokens_than_numbers(gpu_ctx):
    """What no table holds is counted nowhere sensible, and written nowhere."""
    for room in (50, 5000):
        pages = c4s.Pages.empty(3, 4, 40, 16)
        off, pos, slot = i32([0] * 4), i32([-9] * room), i32([-9] * room)
        gpu_ctx.pages_grow(pages, i32([2 ** 31 - 1, 7, 2 ** 31 - 1]), off, pos, slot)
        gpu_ctx.pages_grow(pages, i32([2 ** 31 - 1, 7, 2 ** 31 - 1]), off, pos, slot)
        assert pages.lens.tolist() == [2 ** 31 - 1, 14, 2 ** 31 - 1]
        assert pages.block_table.tolist() == [[0, 1, 2, 3], [4, -1, -1, -1], [5, 6, 7, 8]]
        assert pages.refs.tolist() == [1] * 9 + [0] * 31


def test_bits_behind_the_last_page(gpu_ctx):
    """They name no pages."""
    for n_pages in (3, 33, 70, 120, 127):
        pages = c4s.Pages.empty(2, 200, n_pages, 16)
        pages.free_bits.fill_(-1)
        gpu_ctx.pages_grow(pages, i32([16 * 50, 16 * 100]))
        assert sorted(p for p in pages.block_table.flatten().tolist() if p >= 0) == list(range(min(n_pages, 150)))
        assert pages.refs.tolist() == [1] * n_pages and int(pages.missing) == 150 - n_pages


def test_beams_that_part(gpu_ctx):
    """Who copies a shared last page: all but the last of its holders, all of them where one does not go on, nobody
    where it is full."""
    pool = B.Pool(8, 4, 40, 16)
    pages = pool.device()
    _grow(gpu_ctx, pool, pages, [20, 0, 0, 0, 32, 0, 0, 0], False)
    for f in (pool.fork, lambda p, w: gpu_ctx.pages_fork(pages, i32(p), w)):
        f([0] * 8, 4)
    pool.same(pages)
    pairs = _grow(gpu_ctx, pool, pages, [1, 1, 0, 1, 1, 1, 1, 1], True)[3]
    assert [p[0] >= 0 for p in pairs] == [True, True, False, True] + [False] * 4
    pairs = _grow(gpu_ctx, pool, pages, [0, 0, 3, 0, 0, 0, 0, 0], True)[3]
    assert all(p == (-1, -1) for p in pairs)
    for f in (pool.fork, lambda p, w: gpu_ctx.pages_fork(pages, i32(p), w)):
        f([1, 1, 3, 3, 0, 1, 2, 3], 4)
    pairs = _grow(gpu_ctx, pool, pages, None, True)[3]
    assert [p[0] >= 0 for p in pairs] == [True, False, True, False] + [False] * 4


@pytest.mark.parametrize("store", ["bf16", "q8", "q4"])
@pytest.mark.parametrize("heads,dim,page", [(20, 64, 16), (3, 96, 128), (1, 32, 16), (5, 256, 256), (65, 256, 64)])
def test_kv_copy(gpu_ctx, heads, dim, page, store):
    print(f"kv_copy {heads} heads of {dim}, page={page} {store}", flush=True)
    n = 12
    kc = c4s.KvCache.empty(n, heads, page, dim, torch.zeros((1, 1), dtype=I32, device="cuda"), store=store)
    tensors = [t for t in (kc.k, kc.v, kc.k_scale, kc.v_scale) if t is not None]
    g = torch.Generator(device="cuda").manual_seed(dim)
    for t in tensors:
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, generator=g, device="cuda", dtype=torch.uint8))
    want = [t.view(torch.uint8).clone() for t in tensors]
    pairs = [(-1, -1), (2, 7), (2, 9), (0, 0), (11, 1), (3, n), (-1, 4), (n + 3, 5), (6, -1)]
    gpu_ctx.kv_copy(kc, i32(pairs))
    for w, t in zip(want, tensors):
        for a, b in ((2, 7), (2, 9), (11, 1)):
            w[b] = w[a]
        assert torch.equal(w, t.view(torch.uint8))


def test_kv_copy_past_32_bits(gpu_ctx):
    kc = c4s.KvCache.empty(17000, 16, 64, 128, torch.zeros((1, 1), dtype=I32, device="cuda"))
    for t in (kc.k, kc.v):
        t[16998].fill_(3.0)
        t[16990].fill_(1.0)
        t[16997].fill_(2.0)
        t[16999].fill_(2.0)
    gpu_ctx.kv_copy(kc, i32([[16990, 16998]]))
    for t in (kc.k, kc.v):
        assert (t[16998] == 1).all() and (t[16997] == 2).all() and (t[16999] == 2).all()


def test_in_a_graph(gpu_ctx):
    """A beam step's calls, captured, replayed with eager work in between: the simulation's state after every one."""
    pool = B.Pool(6, 30, 100, 16)
    pages = pool.device()
    _grow(gpu_ctx, pool, pages, [30, 0, 0, 7, 0, 0], False)
    parent, pairs = i32([0] * 6), torch.empty((6, 2), dtype=I32, device="cuda")
    off, pos = torch.empty(7, dtype=I32, device="cuda"), torch.empty(6, dtype=I32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        gpu_ctx.pages_fork(pages, parent, 3)
        gpu_ctx.pages_grow(pages, None, off, pos, None, pairs)
    r = random.Random(1)
    for step in range(25):
        p = [0] * 6 if step == 0 else [r.randrange(3) for _ in range(6)]
        parent.copy_(i32(p))
        graph.replay()
        torch.cuda.synchronize()
        pool.fork(p, 3)
        want = pool.grow(None, True)
        pool.same(pages)
        assert [tuple(x) for x in pairs.tolist()] == want[3] and pos.tolist() == want[1] and off.tolist() == want[0]


def test_nothing_and_refusals(gpu_ctx):
    z = lambda *s, t=I32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    none = c4s.Pages(z(0, 3), z(0), z(6), z(1), 16)
    gpu_ctx.pages_grow(none)
    gpu_ctx.pages_trim(none, z(0))
    gpu_ctx.pages_fork(none, z(0), 2)
    flat = c4s.Pages(z(2, 0), z(2), z(6), z(1), 16, z(1))      # a table without entries
    gpu_ctx.pages_grow(flat, i32([20, 0]))
    gpu_ctx.pages_fork(flat, i32([0, 0]), 2)
    assert flat.lens.tolist() == [20, 20] and flat.missing.tolist() == [2]
    gpu_ctx.pages_trim(flat, i32([5, 30]))
    assert flat.lens.tolist() == [15, 0]
    for args, what in (((z(2, 3), z(2), z(6), z(1), 24), "page_size"), ((z(4097, 1), z(4097), z(6), z(1), 16), "4096"),
                       ((z(1, 131073), z(1), z(6), z(1), 16), "max_pages"), ((z(1, 1), z(1), z(0), z(0), 16), "n_pages")):
        bad = c4s.Pages(*args)
        for call in (lambda: gpu_ctx.pages_grow(bad), lambda: gpu_ctx.pages_trim(bad, bad.lens), lambda: gpu_ctx.pages_fork(bad, bad.lens, 1)):
            with pytest.raises(c4s.C4SError, match=f"code 1.*{what}"):
                call()
    p = c4s.Pages.empty(4, 3, 9, 16)
    with pytest.raises(c4s.C4SError, match="code 1.*need rows_off"):
        gpu_ctx.pages_grow(p, z(4), row_pos=z(5))
    for width in (0, 3, 33):
        with pytest.raises(c4s.C4SError, match="code 1.*width"):
            gpu_ctx.pages_fork(p, z(4), width)
    odd = c4s.Pages(z(4, 3), z(4), z(9 * 32), z(10)[1:], 16)
    with pytest.raises(c4s.C4SError, match="code 1.*16-byte"):
        gpu_ctx.pages_grow(odd)
    for bad in (lambda: gpu_ctx.pages_grow(p, z(3)), lambda: gpu_ctx.pages_grow(p, rows_off=z(4)), lambda: gpu_ctx.pages_grow(p, copies=z(4)),
                lambda: gpu_ctx.pages_trim(p, z(4, t=torch.int64)), lambda: gpu_ctx.pages_fork(p, z(5), 2),
                lambda: c4s.Pages(z(4, 3), z(3), z(9), z(1), 16), lambda: c4s.Pages(z(4, 3), z(4), z(33), z(1), 16)):
        with pytest.raises(ValueError):
            bad()
    kc = c4s.KvCache.empty(4, 2, 16, 64, z(1, 1))
    gpu_ctx.kv_copy(kc, z(0, 2))
    with pytest.raises(c4s.C4SError, match="code 1.*65535"):
        gpu_ctx.kv_copy(kc, z(65536, 2))
    with pytest.raises(c4s.C4SError, match="code 1.*8-byte"):
        gpu_ctx.kv_copy(kc, z(5)[1:].view(2, 2))
    with pytest.raises(ValueError):
        gpu_ctx.kv_copy(kc, z(4))
    torch.cuda.synchronize()
