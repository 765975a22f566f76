"""Pages, the cache's writer and the attention of chunks together, as a server calls them."""
from __future__ import annotations

import random

import pytest

from tests.gpu_util import print_case
from tests.test_gpu_kv8_chunk import attend64

pytestmark = pytest.mark.gpu


class Server:
    """Two layers' caches over one table; the keys and values that every row was given are kept beside it."""

    def __init__(self, dev, pages, rows, width, page, hq, hkv, d, seed=0):
        import torch

        from neurova_amd.attention import KV8Cache
        from neurova_amd.pages import KV8Pages

        self.dev, self.page, self.hq, self.hkv, self.d = dev, page, hq, hkv, d
        self.caches = [KV8Cache(pages, hkv, d, page_size=page, device=dev) for _ in range(2)]
        self.pages = KV8Pages(pages, rows, width * page, page_size=page, caches=self.caches, device=dev)
        self.given = [[torch.zeros((2, 0, hkv, d), dtype=torch.float16, device=dev) for _ in range(2)] for _ in range(rows)]
        self.g = torch.Generator(device=dev)
        self.g.manual_seed(seed)

    def i32(self, x):
        import torch

        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def step(self, rows, new):
        import torch

        assert int(self.pages.extend(self.i32(rows), self.i32(new))) == 0
        at = self.i32(rows)
        table, lens = self.pages.page_table.index_select(0, at), self.pages.seq_lens.index_select(0, at)
        starts = self.i32([0] + torch.tensor(new).cumsum(0).tolist())
        for i, cache in enumerate(self.caches):
            qkv = torch.randn((sum(new), self.hq + 2 * self.hkv, self.d), device=self.dev, generator=self.g).half()
            q, k, v = qkv.split([self.hq, self.hkv, self.hkv], dim=1)
            cache.append(None, k, v, table, lens, starts)
            out = cache.attend(q, table, lens, starts)
            first = 0
            for row, n in zip(rows, new):
                kv = torch.stack([k[first:first + n], v[first:first + n]])
                self.given[row][i] = torch.cat([self.given[row][i], kv], dim=1)
                self.check(i, row, q[first:first + n].double(), out[first:first + n].double())
                first += n

    def check(self, i, row, q, out):
        """The row's pages hold what it was given, within the steps of their scales, and its newest tokens attend to all of it."""
        import torch

        cache, n = self.caches[i], self.given[row][i].shape[1]
        assert int(self.pages.seq_lens[row]) == n
        page = self.pages.page_table[row, :-(-n // self.page)].long()
        assert (page >= 0).all()
        ck = cache.k_cache[page].double().transpose(1, 2).reshape(-1, self.hkv, self.d)[:n]
        cv = cache.v_cache[page].double().permute(0, 3, 1, 2).reshape(-1, self.hkv, self.d)[:n]
        ks, vs = (t[page].double().repeat_interleave(self.page, 0)[:n] for t in (cache.k_scale, cache.v_scale))
        for codes, scale, given in ((ck, ks, self.given[row][i][0]), (cv, vs, self.given[row][i][1])):
            # a value is rounded once when it is stored and once more each time that its page's
            # scale grows: by at most half a step each, and with normally distributed values a
            # page's largest grows a few times, as its tokens arrive, to less than twice its size
            assert ((codes * scale[..., None] - given.double()).abs() <= 6 * scale[..., None]).all(), (i, row)
        sees = torch.arange(n, device=self.dev) <= torch.arange(n - len(q), n, device=self.dev)[:, None]
        for h in range(self.hq):
            g = h // (self.hq // self.hkv)
            want, bound = attend64(q[:, h], ck[:, g], ks[:, g], cv[:, g], vs[:, g], self.d ** -0.5, sees)
            assert ((out[:, h] - want).abs() <= bound).all(), (i, row, h)


@pytest.mark.parametrize("page,hq,hkv,d", [(16, 6, 2, 64), (32, 5, 1, 128), (64, 4, 2, 256)])
def test_pieces_branches_cuts_and_compaction(dev, page, hq, hkv, d):
    print_case("serving", page, hq, hkv, d)
    rng = random.Random(page)
    s = Server(dev, 60, 12, 9, page, hq, hkv, d, seed=page)
    s.step([0, 1], [page + 5, 7])                           # prompts in pieces
    s.step([1, 0], [2 * page, 3])
    s.pages.fork(s.i32([0, 0, 1, 0]), s.i32([2, 3, 4, 5]), s.i32([page + 8, page + 8, 2 * page + 7, page]))
    for child, parent, n in ((2, 0, page + 8), (3, 0, page + 8), (4, 1, 2 * page + 7), (5, 0, page)):
        s.given[child] = [x[:, :n].clone() for x in s.given[parent]]
    s.step([2, 3, 4], [1, 4, 1])                            # their shared last pages are copied
    s.step([0, 5, 1, 4], [1, 2, 40, 9])                     # beside a piece of another prompt
    for _ in range(3):
        rows = rng.sample(range(6), 4)
        s.step(rows, [rng.choice([1, 1, 3, 20]) for _ in rows])
        cut = rng.sample(rows, 2)                           # drafts that were rejected
        keep = [int(s.pages.seq_lens[r]) - 1 for r in cut]
        s.pages.free(s.i32(cut), s.i32(keep))
        for r, n in zip(cut, keep):
            s.given[r] = [x[:, :n] for x in s.given[r]]
    s.pages.free(s.i32([0, 3]))
    for r in (0, 3):
        s.given[r] = [x[:, :0] for x in s.given[r]]
    used = int(s.pages.compact())
    assert used == int((s.pages.refs > 0).sum()) == int(s.pages.page_table.max()) + 1
    s.step([5, 4, 2, 1, 3], [2, 1, 1, 5, 30])               # over moved pages, and a new prompt among them


def test_the_example_runs(dev, capsys):
    from examples import serving

    print_case("serving-example")
    assert serving.main(["--prompts", "300", "41", "90", "--piece", "128", "--answers", "3", "--steps", "4"]) == 0
    assert "finite: True" in capsys.readouterr().out
