"""The operators on pages against a model of the table in plain Python: every entry, length, count and copied byte equal."""
from __future__ import annotations

import random

import pytest

from tests.gpu_util import print_case

pytestmark = pytest.mark.gpu


class Model:
    """What ``include/langburst_lowbit.h`` says of the tables, one entry at a time; `was[p]`: whose codes page p holds."""

    def __init__(self, pages, rows, width, page):
        self.p, self.width = page, width
        self.table = [[-1] * width for _ in range(rows)]
        self.lens, self.refs, self.was = [0] * rows, [0] * pages, list(range(pages))

    def need(self, tokens):
        return -(-tokens // self.p)

    def drop(self, page):
        if 0 <= page < len(self.refs):
            self.refs[page] -= 1

    def free(self, rows, keep=None):
        for i, r in enumerate(rows):
            if not 0 <= r < len(self.table):
                continue
            k = max(keep[i], 0) if keep else 0
            for c in range(self.need(k), self.width):
                if self.table[r][c] >= 0:
                    self.drop(self.table[r][c])
                    self.table[r][c] = -1
            self.lens[r] = min(self.lens[r], k)

    def fork(self, parents, children, lens=None):
        old_lens, old = list(self.lens), [list(r) for r in self.table]
        done, named = [], set()
        for i, (a, c) in enumerate(zip(parents, children)):
            ok = 0 <= a < len(old) and 0 <= c < len(old) and old_lens[c] <= 0 and c not in named
            named.add(c)
            done.append(int(ok))
            if ok:
                n = max(old_lens[a], 0)
                if lens:
                    n = min(n, max(lens[i], 0))
                n = min(n, self.width * self.p)
                for j in range(self.need(n)):
                    page = old[a][j]
                    real = 0 <= page < len(self.refs)
                    self.table[c][j] = page if real else -1
                    if real:
                        self.refs[page] += 1
                self.lens[c] = n
        return done

    def extend(self, rows, add, layers=True):
        seen, todo, sharers = set(), [], {}
        for r, n in zip(rows, add):
            if not 0 <= r < len(self.table) or r in seen:
                continue
            seen.add(r)
            if n <= 0:
                continue
            length = max(self.lens[r], 0)
            if length + n > self.width * self.p:
                return -1
            copy = None
            if length % self.p:
                x = self.table[r][length // self.p]
                if 0 <= x < len(self.refs) and self.refs[x] > 1:
                    rank = sharers.get(x, 0)
                    sharers[x] = rank + 1
                    if rank < self.refs[x] - 1:
                        copy = x
            todo.append((r, length, n, copy, self.need(length + n) - self.need(length)))
        if any(t[3] is not None for t in todo) and not layers:
            return -2
        free = [i for i, x in enumerate(self.refs) if x <= 0]
        total = sum(t[4] + (t[3] is not None) for t in todo)
        if total > len(free):
            return total - len(free)
        for r, length, n, copy, fresh in todo:
            if copy is not None:
                to = free.pop(0)
                self.table[r][length // self.p] = to
                self.refs[to], self.was[to] = 1, self.was[copy]
                self.refs[copy] -= 1
            for j in range(fresh):
                to = free.pop(0)
                self.table[r][self.need(length) + j] = to
                self.refs[to] = 1
            self.lens[r] = length + n
        return 0

    def compact(self):
        used = sum(x > 0 for x in self.refs)
        src = [i for i, x in enumerate(self.refs) if x > 0 and i >= used]
        dst = [i for i, x in enumerate(self.refs) if x <= 0 and i < used]
        move = dict(zip(src, dst))
        for a, b in move.items():
            self.refs[b], self.refs[a], self.was[b] = self.refs[a], 0, self.was[a]
        self.table = [[move.get(x, x) for x in r] for r in self.table]
        return used


class Pool:
    """The same on the GPU: a KV8Pages over caches whose every page has codes and scales of its own."""

    def __init__(self, dev, pages, rows, width, page, layers=2, heads=2, dim=64, seed=0):
        import torch

        from neurova_amd.attention import KV8Cache
        from neurova_amd.pages import KV8Pages

        self.dev = dev
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        self.caches = [KV8Cache(pages, heads, dim, page_size=page, device=dev) for _ in range(layers)]
        for c in self.caches:
            for name in ("k_cache", "v_cache"):
                getattr(c, name).random_(-127, 128, generator=g)
            for name in ("k_scale", "v_scale"):
                getattr(c, name).uniform_(generator=g)
        self.first = [[t.clone() for t in c._buffers()] for c in self.caches]
        self.pages = KV8Pages(pages, rows, width * page, page_size=page, caches=self.caches, device=dev)
        self.model = Model(pages, rows, width, page)

    def i32(self, x):
        import torch

        return None if x is None else torch.tensor(x, dtype=torch.int32, device=self.dev)

    def same(self, what=""):
        import torch

        m, p = self.model, self.pages
        assert p.seq_lens.tolist() == m.lens, what
        assert p.refs.tolist() == m.refs, what
        assert p.page_table.tolist() == m.table, what
        was = torch.tensor(m.was, dtype=torch.int64, device=self.dev)
        held = torch.tensor([x > 0 for x in m.refs], dtype=torch.bool, device=self.dev)
        for c, first in zip(self.caches, self.first):
            for now, then in zip(c._buffers(), first):
                assert torch.equal(now[held], then[was][held]), what

    def extend(self, rows, add):
        got = int(self.pages.extend(self.i32(rows), self.i32(add)))
        want = self.model.extend(rows, add)
        assert got == want, (rows, add)
        return want

    def fork(self, parents, children, lens=None):
        done = self.i32([7] * len(parents))
        self.pages.fork(self.i32(parents), self.i32(children), self.i32(lens), done)
        assert done.tolist() == self.model.fork(parents, children, lens)

    def free(self, rows, keep=None):
        self.pages.free(self.i32(rows), self.i32(keep))
        self.model.free(rows, keep)

    def compact(self):
        assert int(self.pages.compact()) == self.model.compact()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("seed", range(3))
def test_any_sequence_of_calls_matches_the_model(dev, page, seed):
    rng = random.Random(seed * 1000 + page)
    rows, width = rng.choice([(5, 6), (40, 9), (130, 4)])
    print_case("pages-any", page, seed, rows, width)
    pool = Pool(dev, rng.choice([17, 64, 333]), rows, width, page, layers=rng.choice([1, 2, 5]), heads=rng.choice([1, 3]),
                dim=rng.choice([64, 128, 256]), seed=seed)
    for step in range(40):
        n = rng.randint(1, rows)
        some = [rng.randint(-1, rows) if rng.random() < 0.1 else rng.randrange(rows) for _ in range(n)]  # named twice, and outside
        what = rng.choice(["extend", "extend", "extend", "fork", "fork", "free", "compact"])
        if what == "extend":
            pool.extend(some, [rng.choice([-1, 0, 1, 1, 2, page, rng.randint(0, 2 * page)]) for _ in some])
        elif what == "fork":
            lens = None if rng.random() < 0.5 else [rng.choice([-3, 0, page, rng.randint(0, width * page)]) for _ in some]
            pool.fork([rng.randrange(rows) for _ in some], some, lens)
        elif what == "free":
            pool.free(some, None if rng.random() < 0.4 else [rng.randint(-1, width * page) for _ in some])
        else:
            pool.compact()
        pool.same((step, what))


def test_a_full_pool_and_a_full_row_refuse_the_whole_call(dev):
    print_case("pages-full")
    pool = Pool(dev, 10, 4, 8, 16)
    assert pool.extend([0, 1], [100, 20]) == 0           # seven pages and two
    assert pool.extend([2, 3], [16, 40]) == 3            # four are needed, one is left
    pool.same()
    assert pool.extend([0, 2], [29, 1]) == -1            # past the table's 128 tokens
    assert pool.extend([0], [12]) == 0 and pool.extend([2], [16]) == 0
    pool.same()
    pool.fork([1], [3])
    assert pool.extend([1], [1]) == 1                    # its last page is shared, and there is none for a copy
    pool.same()
    pool.free([0], [40])
    assert pool.extend([1, 3], [1, 1]) == 0              # a copy for one of the two
    pool.same()


def test_shared_pages_are_copied_for_all_but_the_last_holder(dev):
    print_case("pages-shared")
    pool = Pool(dev, 64, 12, 8, 16, layers=3)
    pool.extend([3], [37])
    pool.fork([3] * 5, [0, 1, 2, 4, 5], [37, 37, 32, 33, 20])
    pool.extend([0, 1, 2], [1, 30, 1])                   # three holders of the last page stay outside the call
    pool.same("outside")
    pool.extend([5, 4, 3], [1, 1, 1])                    # and now the last keeps it
    pool.same("last")
    pool.fork([5, 5], [6, 7], [32, 21])                  # a whole page, and a part
    pool.extend([7, 6, 5], [1, 1, 1])
    pool.same("part")


def test_without_caches_pages_are_counted_and_copies_refused(dev):
    import torch

    from neurova_amd.pages import KV8Pages

    print_case("pages-no-caches")
    p = KV8Pages(32, 4, 128, page_size=16, device=dev)
    m = Model(32, 4, 8, 16)
    one = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    assert int(p.extend(one([2]), 20)) == m.extend([2], [20]) == 0
    p.fork(one([2]), one([0]))
    m.fork([2], [0])
    assert int(p.extend(one([0]), 1)) == m.extend([0], [1], layers=False) == -2
    assert int(p.extend(one([0]), 0)) == m.extend([0], [0], layers=False) == 0
    p.free(one([2]))
    m.free([2])
    assert int(p.extend(one([0]), 40)) == m.extend([0], [40], layers=False) == 0
    assert int(p.compact()) == m.compact()
    assert p.page_table.tolist() == m.table and p.refs.tolist() == m.refs and p.seq_lens.tolist() == m.lens


@pytest.mark.parametrize("pages,rows,width", [(40000, 4096, 9), (70001, 3, 20000), (1, 1, 1), (16384, 100, 150), (5, 2, 0), (3000, 9000, 3), (0, 3, 2)])
def test_large_and_small_pools(dev, pages, rows, width):
    """As many rows as a call takes, rows of many pages, and pools whose ends fall inside what is looked at together."""
    print_case("pages-large", pages, rows, width)
    rng = random.Random(pages)
    pool = Pool(dev, pages, rows, width, 16, layers=1, heads=1, seed=1)
    order = rng.sample(range(rows), min(rows, 4096))
    order[5:7] = order[:2] if len(order) > 9 else order[5:7]    # two rows named twice
    most = min(width * 16, pages * 16 // max(rows, 1))
    pool.extend(order, [rng.randint(0, most) for _ in order])
    pool.free(order[::3])
    pool.free(order[1::3], [rng.randint(0, most) for _ in order[1::3]])
    pool.fork(order[2::3][:len(order[::3])], order[::3][:len(order[2::3])])
    pool.extend(order[::-1], [rng.choice([0, 1]) for _ in order])
    pool.same()
    pool.compact()
    pool.same()
    pool.extend([0], [min(most, 5)])
    pool.same()


def test_the_layers_of_a_large_model(dev):
    """More layers than one launch takes, pages of more and less than a workgroup's piece."""
    print_case("pages-layers")
    for heads, dim, page, layers in ((1, 64, 16, 70), (8, 256, 32, 33), (3, 128, 64, 2)):
        pool = Pool(dev, 24, 6, 6, page, layers=layers, heads=heads, dim=dim)
        pool.extend([0, 1], [2 * page + 3, page])
        pool.fork([0, 0], [2, 3])
        pool.extend([2, 3, 0], [1, 1, 1])
        pool.same()
        pool.free([1, 2])
        pool.compact()
        pool.same()


def test_copies_between_pages(dev):
    import torch

    import langburst_cuda as lc
    from neurova_amd.pages import copy_pages, kv8_layers

    print_case("pages-copy")
    pool = Pool(dev, 50, 1, 1, 32, layers=3, heads=3, dim=128)
    src, dst = [4, 9, 4, -1, 7, 50, 12], [11, 49, 0, 13, 50, 14, 12]   # outside the pool, and onto itself: left out
    copy_pages(pool.caches, pool.i32(src), pool.i32(dst))
    want = list(range(50))
    for a, b in zip(src, dst):
        if 0 <= a < 50 and 0 <= b < 50:
            want[b] = a
    for c, first in zip(pool.caches, pool.first):
        for now, then in zip(c._buffers(), first):
            assert torch.equal(now, then[torch.tensor(want, device=dev)])
    layers = kv8_layers(pool.caches)
    assert len(layers) == 3
    lc.kv8_copy_pages(layers, pool.i32([]), pool.i32([]))


def test_a_cache_larger_than_32_bit_offsets(dev):
    import torch

    from neurova_amd.pages import copy_pages

    pages = (1 << 32) // (128 * 4 * 256) + 20
    print_case("pages-4GiB", pages)
    pool = Pool(dev, 1, 1, 1, 128, layers=1, heads=4, dim=256)
    c = pool.caches[0]
    old = [t.clone() for t in c._buffers()]
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        t = getattr(c, name)
        setattr(c, name, torch.empty((pages, *t.shape[1:]), dtype=t.dtype, device=dev))
        getattr(c, name)[2] = t[0]
    copy_pages([c], pool.i32([2]), pool.i32([pages - 1]))
    copy_pages([c], pool.i32([pages - 1]), pool.i32([pages - 9]))
    for now, then in zip(c._buffers(), old):
        assert torch.equal(now[pages - 1], then[0]) and torch.equal(now[pages - 9], then[0])


def test_pages_captured_into_a_graph(dev):
    """A server's step, replayed with eager calls between: drafts are cut, pages for the next handed out, ended rows forked anew."""
    import torch

    print_case("pages-graph")
    pool = Pool(dev, 600, 20, 12, 16, layers=2)
    pool.extend([0], [75])
    pool.fork([0] * 10, list(range(1, 11)))
    pool.extend(list(range(11)), [5] * 11)
    rows, keep = pool.i32(list(range(1, 11))), pool.i32([77 + i for i in range(10)])
    last, add, status = pool.i32([0, 0]), pool.i32([3] * 10), pool.i32([9])
    children, used = pool.i32([15, 16]), pool.i32([0])
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            pool.pages.free(rows, keep)
            pool.pages.free(children)
            pool.pages.fork(last, children)
            pool.pages.extend(rows, add, status)
            pool.pages.compact(used)
    torch.cuda.synchronize()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        m = pool.model
        m.free(rows.tolist(), keep.tolist())
        m.free([15, 16])
        m.fork([0, 0], [15, 16])
        assert int(status) == m.extend(rows.tolist(), add.tolist()) == 0
        assert int(used) == m.compact()
        pool.same(i)
        pool.extend([0, 15], [1, 1])  # eager work, and the next replay begins elsewhere
        pool.same(i)


def test_tables_with_strides_another_stream_and_the_c_abi(dev):
    import torch

    from neurova_amd import capi

    print_case("pages-strided")
    pool = Pool(dev, 40, 6, 8, 16)
    wide = torch.full((6, 13), 5, dtype=torch.int32, device=dev)
    view = wide[:, 2:10]
    view.fill_(-1)
    pool.pages.page_table = view
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.extend([1, 4], [50, 33])
        pool.fork([1], [2], [40])
        pool.extend([2, 1], [1, 1])
        pool.free([4])
        pool.compact()
        pool.same()
    torch.cuda.current_stream().wait_stream(side)
    assert (wide[:, :2] == 5).all() and (wide[:, 10:] == 5).all()
    p, m = pool.pages, pool.model
    scratch = torch.empty(max(capi.lib().lb_kv8_pages_extend_scratch_bytes(40), capi.lib().lb_kv8_pages_compact_scratch_bytes(40)),
                          dtype=torch.uint8, device=dev)
    caches, status, done = [c._buffers() for c in pool.caches], pool.i32([0]), pool.i32([0])
    state = (p.page_table, p.seq_lens, p.refs, 16)
    assert capi.kv8_pages_fork(*state, pool.i32([2]), pool.i32([5]), None, done) == 0 and done.tolist() == m.fork([2], [5])
    assert capi.kv8_pages_extend(*state, pool.i32([5]), pool.i32([9]), status, caches, scratch) == 0 and int(status) == m.extend([5], [9])
    pool.same()
    assert capi.kv8_pages_free(*state, pool.i32([1]), pool.i32([3])) == 0
    m.free([1], [3])
    assert capi.kv8_pages_compact(p.page_table, p.refs, 16, status, caches, scratch) == 0 and int(status) == m.compact()
    pool.same()
    free = [i for i, x in enumerate(m.refs) if not x]
    assert capi.kv8_copy_pages(caches, pool.i32([m.table[1][0]]), pool.i32([free[-1]])) == 0
    torch.cuda.synchronize()
    assert torch.equal(pool.caches[1].k_cache[free[-1]], pool.caches[1].k_cache[m.table[1][0]])


def test_refusals(dev):
    import torch

    import langburst_cuda as lc
    from neurova_amd.pages import KV8Pages, kv8_layers

    print_case("pages-refusals")
    pool = Pool(dev, 8, 3, 4, 16)
    p, one = pool.pages, pool.i32([1])
    with pytest.raises(RuntimeError, match="must have 1 entries"):
        p.extend(one, pool.i32([1, 2]))
    with pytest.raises(RuntimeError, match="int32"):
        p.free(one.long())
    with pytest.raises(RuntimeError, match="same device"):
        p.fork(one, one.cpu())
    with pytest.raises(RuntimeError, match="at most 4096"):
        p.free(torch.zeros(4097, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="rows\\] of page_table"):
        lc.kv8_pages_free_out(p.page_table, p.seq_lens[:2], p.refs, 16, one, None)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        lc.kv8_pages_free_out(p.page_table, p.seq_lens, torch.zeros(9, dtype=torch.int32, device=dev)[1:], 16, one, None)
    with pytest.raises(RuntimeError, match="that refs counts"):
        lc.kv8_pages_extend_out(p.page_table, p.seq_lens, p.refs, 32, one, one, one.clone(), p.layers)
    with pytest.raises(RuntimeError, match="code 1 "):
        lc.kv8_pages_free_out(p.page_table, p.seq_lens, p.refs, 17, one, None)
    other = Pool(dev, 9, 3, 4, 16)
    with pytest.raises(RuntimeError, match="that refs counts"):
        lc.kv8_pages_compact_out(p.page_table, p.refs, one.clone(), other.pages.layers)
    with pytest.raises(RuntimeError, match="same shape"):
        kv8_layers([pool.caches[0], other.caches[0]])
    with pytest.raises(ValueError, match="page_size"):
        KV8Pages(8, 1, 64, page_size=20, device=dev)
    pool.same()


@pytest.mark.parametrize("children, width", [(128, 16), (129, 16), (1, 2048), (1, 2049), (2047, 1), (700, 3)])
def test_forks_of_few_and_many_entries(dev, children, width):
    """One launch up to 2048 entries, two above; with parts of pages, rows named twice, outside, and holding tokens."""
    print_case("pages-fork-entries", children, width)
    rng = random.Random(children + width)
    pool = Pool(dev, 2 * width + 5, children + 3, width, 16, layers=1, heads=1)
    assert pool.extend([0, 1], [width * 16, max(width * 16 - 9, 1)]) == 0
    named = [rng.randrange(2, children + 3) for _ in range(children)]
    named[0] = rng.choice([-1, children + 3, 1])
    parents = [rng.choice([0, 1, 1, 2, -1]) for _ in named]
    pool.fork(parents, named, [rng.choice([0, 1, 15, 16, 17, width * 8, width * 16 + 3]) for _ in named])
    pool.same("first")
    pool.free(named[::2])
    pool.fork(parents[::-1], named[::-1])
    pool.same("second")


def test_rows_of_many_pages(dev):
    """Tables wider than a workgroup's turn, and than a turn of all workgroups of a row: cut, forked, ended."""
    import torch

    from neurova_amd.pages import KV8Pages

    print_case("pages-wide")
    width = 256 * 4096 + 300
    pages = KV8Pages(2 * width, 4, width * 16, page_size=16, device=dev)
    row = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    assert int(pages.extend(row(2), row(width * 16))) == 0
    want = torch.arange(width, dtype=torch.int32, device=dev)
    assert torch.equal(pages.page_table[2], want) and int(pages.refs.sum()) == width
    pages.fork(row(2), row(0), row(width * 16 - 20))
    assert torch.equal(pages.page_table[0][:width - 1], want[:-1]) and int(pages.page_table[0][-1]) == -1
    assert int(pages.refs.sum()) == 2 * width - 1
    pages.free(row(2), row(16 * 300 + 1))
    assert pages.seq_lens.tolist() == [width * 16 - 20, 0, 16 * 300 + 1, 0]
    assert torch.equal(pages.page_table[2][:301], want[:301]) and int(pages.page_table[2][301:].max()) == -1
    assert int(pages.refs.sum()) == width - 1 + 301 and int(pages.refs[width - 1]) == 0
    pages.free(row(0, 2))
    assert not pages.refs.any() and not pages.seq_lens.any() and int(pages.page_table.max()) == -1
