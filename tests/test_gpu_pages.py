"""Pages handed out, shared, freed, moved and copied, against the same in Python; runs of them together."""

from __future__ import annotations

import random

import pytest
import torch

from .paged_reference import Holder

pytestmark = pytest.mark.gpu


def ints(device, values, dtype=torch.int64):
    return torch.tensor(values, device=device, dtype=dtype)


class Cache:
    """A pool of `layers` with its bookkeeping on the device, and a Holder that says what it should be."""

    def __init__(self, device, n_seq, entries, pages, P, layers=2, G=1, D=8):
        from sva_amd import kernels

        self.k, self.device, self.P, self.shape = kernels, device, P, (layers, G, D)
        self.pool = kernels.pages_alloc(pages, G, P, D, device, torch.float32, layers=layers).fill_(float("nan"))
        self.tables = torch.full((n_seq, entries), -1, device=device, dtype=torch.int32)
        self.lens = torch.zeros(n_seq, device=device, dtype=torch.int64)
        self.refs = torch.zeros(pages, device=device, dtype=torch.int32)
        self.model = Holder(n_seq, entries, pages, P)
        self.value = 0

    def grow(self, counts):
        """Reserve, copy, write rows of new values; what is granted as the Holder says."""
        want, pairs = self.model.reserve(counts)
        first, src, dst = self.k.pages_reserve(self.tables, self.lens, self.refs, ints(self.device, counts), self.P)
        assert first.tolist() == want and list(zip(src.tolist(), dst.tolist())) == pairs
        self.k.pages_copy(self.pool, src, dst)
        L, G, D = self.shape
        for b, (a, c) in enumerate(zip(want, counts)):
            if a < 0 or c == 0:
                continue
            rows = [self.value + t for t in range(c)]
            self.value += c
            self.model.rows[b] += rows
            x = ints(self.device, rows, torch.float32)[None, None, :, None].expand(1, G, c, D)
            for layer in range(L):
                self.k.paged_write(x + 0.25 * layer, -x, self.pool[layer], self.tables[b:b + 1], [a])

    def fork(self, sources):
        self.model.fork(sources)
        self.k.pages_fork(self.tables, self.lens, self.refs, ints(self.device, sources), self.P)

    def compact(self):
        pairs, used = self.model.compact()
        src, dst, n = self.k.pages_compact(self.tables, self.refs)
        assert n.tolist() == [used]
        assert list(zip(src.tolist(), dst.tolist())) == pairs + [(-1, -1)] * (len(src) - len(pairs))
        self.k.pages_copy(self.pool, src, dst)

    def check(self):
        held = [t[:-(-n // self.P)] for t, n in zip(self.tables.tolist(), self.lens.tolist())]
        assert self.lens.tolist() == self.model.lens
        assert held == self.model.held
        assert self.refs.tolist() == self.model.refs()
        most = max(self.model.lens)
        for layer in range(self.shape[0]):
            keys, values = self.k.paged_read(self.pool[layer], self.tables, [0] * len(held), most)
            for b, rows in enumerate(self.model.rows):
                want = ints(self.device, rows, torch.float32)[None, :, None]
                assert (keys[b, :, :len(rows)] == want + 0.25 * layer).all() and (values[b, :, :len(rows)] == -want).all()


@pytest.mark.parametrize("seed,n_seq,entries,pages,P", [(1, 1, 3, 2, 16), (2, 5, 6, 17, 16), (3, 8, 4, 40, 32), (4, 40, 9, 200, 16),
                                                        (5, 3, 300, 700, 16), (6, 3, 6000, 9000, 16), (7, 1500, 2, 2000, 16)])
def test_random_steps(device, seed, n_seq, entries, pages, P):
    """Growth that is granted or not, forks of forks, swaps, frees and compactions, in any order."""
    rng = random.Random(seed)
    c = Cache(device, n_seq, entries, pages, P)
    for _ in range(25):
        step = rng.choice(["grow", "grow", "grow", "fork", "fork", "free", "compact"])
        if step == "grow":
            c.grow([rng.choice([0, 0, 1, 1, 2, P, rng.randint(0, P * max(1, entries // 3)), -1]) for _ in range(n_seq)])
        elif step == "fork":
            c.fork([rng.choice([b, b, rng.randrange(n_seq)]) for b in range(n_seq)])
        elif step == "free":
            c.fork([rng.choice([-1, b, b, b, n_seq, -2]) for b in range(n_seq)])
        else:
            c.compact()
        c.check()


def test_many_sequences_and_pages(device):
    """More sequences than a workgroup has threads, more pages than it looks at a time."""
    c = Cache(device, 2500, 4, 40000, 16, layers=1)
    rng = random.Random(3)
    c.grow([rng.randint(0, 2) for _ in range(2500)])
    c.fork([rng.randrange(2500) if rng.random() < 0.5 else b for b in range(2500)])
    model, k = c.model, c.k
    want, pairs = model.reserve([20] * 2500)
    first, src, dst = k.pages_reserve(c.tables, c.lens, c.refs, 20, 16)
    assert first.tolist() == want and list(zip(src.tolist(), dst.tolist())) == pairs
    assert c.refs.tolist() == model.refs() and c.lens.tolist() == model.lens
    sources = [rng.choice([-1, b]) for b in range(2500)]
    c.fork(sources)
    pairs, used = model.compact()
    src, dst, n = k.pages_compact(c.tables, c.refs)
    assert n.tolist() == [used] and list(zip(src.tolist(), dst.tolist()))[:len(pairs)] == pairs
    assert c.refs.tolist() == model.refs()
    assert [t[:-(-n // 16)] for t, n in zip(c.tables.tolist(), c.lens.tolist())] == model.held


def test_rows_of_sequences_without_room(device):
    """A sequence that was given no room writes none of its rows, the second token no more than the first."""
    from sva_amd import kernels as k

    pool = torch.randn(4, 2, 1, 16, 8, device=device)
    tables, lens = ints(device, [[2, -1, -1, -1], [0, -1, -1, -1]], torch.int32), ints(device, [9, 3])
    refs = ints(device, [1, 0, 1, 0], torch.int32)
    first, src, dst = k.pages_reserve(tables, lens, refs, ints(device, [50, 5]), 16)  # three pages, of two; none
    assert first.tolist() == [-1, 3] and lens.tolist() == [9, 8]
    keys = torch.randn(2, 1, 5, 8, device=device)
    want = pool.clone()
    want[0, 0, 0, 3:8], want[0, 1, 0, 3:8] = keys[1, 0], -keys[1, 0]
    k.paged_write(keys, -keys, pool, tables, first)
    assert torch.equal(pool, want)
    got = k.paged_read(pool, tables, first, 5)
    assert (got[0][0] == 0).all() and (got[1][0] == 0).all() and torch.equal(got[0][1], keys[1])
    for far in (2 ** 63 - 2, -2 ** 63):
        k.paged_write(keys, -keys, pool, tables, [far, far])
        assert torch.equal(pool, want) and (k.paged_read(pool, tables, [far, far], 5)[0] == 0).all()


def test_a_full_pool(device):
    """All pages or none: a sequence whose pages are not there changes nothing, one that needs none goes on."""
    c = Cache(device, 4, 8, 6, 16)
    c.grow([16 * 3, 5, 0, 0])       # 4 of 6 pages
    c.grow([0, 3, 40, 16])          # the third asks for 3 pages, the fourth for one more: neither
    assert c.lens.tolist() == [48, 8, 0, 0]
    c.grow([0, 8, 32, 0])           # the second fills its page, the third takes the last two
    c.grow([0, 1, 0, 0])            # none left
    c.check()
    assert (c.refs == 1).all() and c.lens.tolist() == [48, 16, 32, 0]
    c.fork([0, -1, 2, 3])
    c.grow([0, 0, 0, 1])            # the freed page again
    c.check()
    c.grow([129, 0, 0, 0])          # a table of 8 pages is too short
    c.grow([-5, 0, 0, 0])
    c.check()


def test_every_holder_of_a_shared_page_leaves_it(device):
    c = Cache(device, 3, 4, 12, 16)
    c.grow([20, 0, 0])
    c.fork([0, 0, 0])
    c.grow([1, 1, 1])  # three new last pages; the old one is free again
    c.check()
    assert c.refs.tolist()[:5] == [3, 0, 1, 1, 1]
    c.grow([16, 0, 0])
    c.check()
    assert int(c.tables[0, 2]) == 1


def test_stale_entries_and_bad_numbers(device):
    """Entries behind a length, or outside the pool, are nobody's; compaction leaves those it does not move."""
    from sva_amd import kernels as k

    tables = ints(device, [[5, 2, 7, -1], [3, 900, -4, 6]], torch.int32)
    lens, refs = ints(device, [32, 48]), ints(device, [0, 1, 1, 1, 0, 1, 0, 0], torch.int32)
    k.pages_fork(tables, lens, refs, ints(device, [1, 1]), 16)  # row 0 held 5 and 2; row 1: 3, and two that are no pages
    assert tables.tolist() == [[3, 900, -4, -1], [3, 900, -4, 6]] and lens.tolist() == [48, 48]
    assert refs.tolist() == [0, 1, 0, 2, 0, 0, 0, 0]
    src, dst, used = k.pages_compact(tables, refs)  # (page 1 is held by nobody in the tables, but counted)
    assert used.tolist() == [2] and src.tolist() == [3, -1, -1, -1] and dst.tolist() == [0, -1, -1, -1]
    assert tables.tolist() == [[0, 900, -4, -1], [0, 900, -4, 6]] and refs.tolist() == [2, 1, 0, 0, 0, 0, 0, 0]
    first, src, dst = k.pages_reserve(tables, ints(device, [-1, 10 ** 12]), refs, 1, 16)
    assert first.tolist() == [-1, -1] and src.tolist() == dst.tolist() == [-1, -1]


def test_copies(device):
    """Several layers, pages of odd sizes, sources named twice, pairs outside the pool, long lists that are mostly empty."""
    from sva_amd import kernels as k

    for shape, dtype in (((3, 9, 2, 3, 16, 64), torch.bfloat16), ((9, 2, 1, 16, 8), torch.float32), ((2, 9, 2, 2, 64, 136), torch.float16)):
        pool = torch.randn(shape, device=device).to(dtype)
        want = pool.clone()
        src, dst = [4, -1, 4, 0, 9, 3], [7, 2, 8, 1, 0, -1]
        at = lambda p, i: p[:, i] if len(shape) == 6 else p[i]  # noqa: E731
        for a, b in ((4, 7), (4, 8), (0, 1)):
            at(want, b).copy_(at(want, a))
        k.pages_copy(pool, ints(device, src, torch.int32), ints(device, dst, torch.int32))
        assert torch.equal(pool, want)
    pool = torch.randn(50, 2, 1, 16, 8, device=device)
    want = pool.clone()
    want[40:] = want[:10]
    src, dst = (torch.full((70001,), -1, device=device, dtype=torch.int32) for _ in range(2))
    places = torch.arange(10, device=device) * 7000 + 1
    src[places], dst[places] = torch.arange(10, device=device).int(), torch.arange(40, 50, device=device).int()
    k.pages_copy(pool, src, dst)
    assert torch.equal(pool, want)
    k.pages_copy(pool, src[:0], dst[:0])
    by_page = torch.randn(5, 4, 2, 1, 16, 8, device=device)  # pages before layers
    want = by_page.clone()
    want[3] = want[1]
    k.pages_copy(by_page.transpose(0, 1), ints(device, [1], torch.int32), ints(device, [3], torch.int32))
    assert torch.equal(by_page, want)


def test_empty_pools(device):
    from sva_amd import kernels as k

    none = torch.zeros(0, device=device, dtype=torch.int32)
    tables, lens = torch.full((2, 3), -1, device=device, dtype=torch.int32), ints(device, [0, 0])
    assert k.pages_reserve(tables, lens, none, 1, 16)[0].tolist() == [-1, -1]
    k.pages_fork(tables, lens, none, ints(device, [1, 0]), 16)
    assert k.pages_compact(tables, none)[2].tolist() == [0]
    for n in (0, 3):  # one page
        src, dst, used = k.pages_compact(tables, ints(device, [n], torch.int32))
        assert used.tolist() == [min(n, 1)] and src.shape == dst.shape == (0,)
    refs = ints(device, [0, 1, 0], torch.int32)
    assert k.pages_compact(tables[:0], refs)[2].tolist() == [1] and refs.tolist() == [1, 0, 0]


def test_a_step_in_a_graph(device):
    """Reserve, copy, write and attend captured once and replayed, against the same steps outside a graph."""
    from sva_amd import kernels as k

    def state():
        pool = k.pages_alloc(64, 2, 16, 64, device, torch.float32).zero_()
        tables = torch.full((4, 8), -1, device=device, dtype=torch.int32)
        lens, refs = torch.zeros(4, device=device, dtype=torch.int64), torch.zeros(64, device=device, dtype=torch.int32)
        k.pages_reserve(tables, lens, refs, ints(device, [30, 0, 7, 0]), 16)
        k.pages_fork(tables, lens, refs, ints(device, [0, 0, 2, 2]), 16)
        return pool, tables, lens, refs

    rows, q = torch.zeros(2, 4, 2, 1, 64, device=device), torch.zeros(4, 4, 1, 64, device=device)

    def step(pool, tables, lens, refs):
        first, src, dst = k.pages_reserve(tables, lens, refs, 1, 16)
        k.pages_copy(pool, src, dst)
        k.paged_write(rows[0], rows[1], pool, tables, first)
        return k.paged_attention(q, pool, tables, lens, 0.125)

    a, b = state(), state()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*[x.clone() for x in a])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*a)
    gen = torch.Generator(device=device).manual_seed(0)
    for i in range(40):
        rows.normal_(generator=gen)
        q.normal_(generator=gen)
        graph.replay()
        want = step(*b)
        assert torch.equal(out, want), i
        if i % 7 == 0:
            torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and a[2].tolist() == [70, 70, 47, 47]
