"""The attention operators against 64-bit oracles: the 8-bit cache's writer and reader, and prompts.

Tolerances, set before any run:

* rotated rows are fp16 roundings of fp32 results: 2^-11 of the value plus
  2^-22 of the pair's length and 2^-25 (fp16 subnormals);
* a stored value is within half a step (its page's scale) of the value it
  stands for, a rescaled one within half a new step of the old value; scales
  are max / 127 to 2^-21;
* attention outputs: the output's rounding 2^-11 |o|, the weights' error times
  sum p |v|, and 2^-25 for subnormals.  A weight's error is twice that of its
  score in fp32 (numerator and denominator) plus the hardware exponential and
  the sums (2^-18); prompts round it to fp16 too (2^-11, and 2^-25 of the
  largest weight 2^7 times smaller for tiny ones).
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import attention_oracle as A
from tests.gpu_util import print_case

pytestmark = pytest.mark.gpu


def _gen(dev, seed):
    import torch

    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


# ------------------------------------------------------------------ append ---

class AppendCase:
    """A cache with random contents, `held` tokens per sequence before the call and `news` new ones."""

    def __init__(self, dev, held, news, hq, hkv, d, p, rot, seed=0, strided=False, positions=None, uniform=False):
        import torch

        from neurova_amd.attention import rotation_table

        g = _gen(dev, seed)
        self.held, self.news, self.hq, self.hkv, self.d, self.p, self.rot = held, news, hq, hkv, d, p, rot
        tokens = sum(news)
        wide = hq + 2 * hkv
        if strided:  # heads of a fused projection with a gap after every head
            qkv = torch.randn((tokens, wide + 1, 2 * d), device=dev, generator=g).half()[:, 1:, :d]
        else:
            qkv = torch.randn((tokens, wide, d), device=dev, generator=g).half()
        qkv[:, :, 0] *= 6  # an outlier channel
        self.q, self.k, self.v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        lens = [h + n for h, n in zip(held, news)]
        width = max([1] + [-(-n // p) for n in lens]) + 1
        pool = sum(-(-n // p) for n in lens) + 2
        order = torch.randperm(pool, device="cpu").tolist()
        table = np.full((len(held), width), -7, dtype=np.int32)
        for b, n in enumerate(lens):
            for j in range(-(-n // p)):
                table[b, j] = order.pop()
        self.lens, self.table_np = lens, table
        self.table = torch.from_numpy(table).to(dev)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.starts = None if uniform else torch.tensor(np.cumsum([0] + news), dtype=torch.int32, device=dev)
        self.k_cache = torch.randint(-127, 128, (pool, hkv, p, d), dtype=torch.int8, device=dev, generator=g)
        self.v_cache = torch.randint(-127, 128, (pool, hkv, d, p), dtype=torch.int8, device=dev, generator=g)
        # half of the held pages have scales that the new tokens exceed
        self.k_scale = torch.rand((pool, hkv), device=dev, generator=g) * 0.06 + 1e-3
        self.v_scale = torch.rand((pool, hkv), device=dev, generator=g) * 0.06 + 1e-3
        self.rotation = rotation_table(positions or max(lens + [1]), rot, device=dev) if rot else None
        self.before = [t.clone() for t in (self.k_cache, self.v_cache, self.k_scale, self.v_scale)]

    def run(self, ops, interleaved, q_out=None, k_out=None):
        import torch

        q_out = torch.full((sum(self.news), self.hq, self.d), 7.0, dtype=torch.float16, device=self.q.device) if q_out is None else q_out
        ops.kv8_append_out(self.q, self.k, self.v, self.k_cache, self.v_cache, self.k_scale, self.v_scale, self.table,
                           self.seq_lens, self.starts, self.rotation, q_out, k_out, interleaved)
        torch.cuda.synchronize()
        return q_out

    def check(self, q_out, interleaved, k_out=None):
        rot = None if self.rotation is None else _np(self.rotation)
        q, k, v = _np(self.q), _np(self.k), _np(self.v)
        kb, vb, ksb, vsb = (_np(t) for t in self.before)
        ka, va, ksa, vsa = (_np(t) for t in (self.k_cache, self.v_cache, self.k_scale, self.v_scale))
        vb, va = vb.transpose(0, 1, 3, 2), va.transpose(0, 1, 3, 2)
        p, at, touched = self.p, 0, set()

        def turned(x, pos):
            return np.array(x) if rot is None else A.rotate(x, rot[pos, :self.rot // 2], rot[pos, self.rot // 2:], interleaved)

        def near(got, want, what):
            size = np.abs(want).max() + 1
            assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * size + 2.0 ** -25).all(), what

        for b, (h, n) in enumerate(zip(self.held, self.news)):
            kr = np.stack([turned(k[at + i], h + i) for i in range(n)]) if n else np.zeros((0, self.hkv, self.d))
            for i in range(n):
                near(_np(q_out[at + i]), turned(q[at + i], h + i), (b, i))
                if k_out is not None:
                    near(_np(k_out[at + i]), kr[i], (b, i, "k"))
            for page in range(h // p, -(-(h + n) // p)) if n else []:
                lo, hi = max(h, page * p), min(h + n, (page + 1) * p)
                cell, old = self.table_np[b, page], lo - page * p
                touched.add(int(cell))
                for new, cb, ca, sb, sa in ((kr, kb, ka, ksb, ksa), (v[at:at + n], vb, va, vsb, vsa)):
                    x = new[lo - h:hi - h].transpose(1, 0, 2)
                    need = np.abs(x).max((1, 2)) / 127
                    want = np.maximum(need, sb[cell]) if old else need
                    assert np.allclose(sa[cell], want, rtol=2.0 ** -21, atol=0), (b, page)
                    step = sa[cell][:, None, None]
                    got = ca[cell][:, old:old + hi - lo] * step
                    assert (np.abs(got - x) <= 0.5 * step * (1 + 1e-4)).all(), (b, page, "new")
                    was = cb[cell][:, :old] * sb[cell][:, None, None]
                    grew = (sa[cell] != sb[cell])[:, None, None]
                    diff = np.abs(ca[cell][:, :old] * step - was)
                    assert (diff <= np.where(grew, 0.5 * step * (1 + 1e-4), 0)).all(), (b, page, "old")
                    # slots after the sequence's end keep their codes
                    if hi < (page + 1) * p:
                        assert np.array_equal(ca[cell][:, hi - page * p:], cb[cell][:, hi - page * p:])
            at += n
        rest = [i for i in range(len(ka)) if i not in touched]
        for a, c in ((ka, kb), (va, vb), (ksa, ksb), (vsa, vsb)):
            assert np.array_equal(a[rest], c[rest])


APPEND = [
    # held, news, heads_q, heads_kv, d, page, rot, interleaved, uniform
    ([0], [1], 1, 1, 64, 16, 64, False, True),
    ([5, 16, 31, 100], [1, 1, 1, 1], 6, 2, 128, 16, 128, True, True),
    ([15, 0, 62], [3, 3, 3], 4, 4, 256, 32, 64, False, True),
    ([7, 64, 127], [2, 2, 2], 5, 1, 64, 128, 32, True, True),
    ([0, 3, 0, 40], [33, 1, 0, 90], 8, 2, 128, 32, 96, False, False),
    ([0, 0], [17, 300], 6, 1, 256, 64, 256, True, False),
    ([129], [257], 2, 2, 128, 128, 16, False, False),
    ([11, 1], [5, 31], 3, 3, 64, 16, 0, False, False),
    ([0] * 70, [1, 2] * 35, 2, 1, 64, 16, 64, False, False),
    ([1000], [700], 40, 8, 128, 16, 128, True, False),
    ([30, 95], [64, 64], 3, 1, 256, 128, 128, False, True),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("strided", [False, True])
def test_append_matches_the_definition(dev, case, strided):
    import langburst_cuda as lc
    import torch

    held, news, hq, hkv, d, p, rot, inter, uniform = APPEND[case]
    print_case("append", *APPEND[case], strided)
    c = AppendCase(dev, held, news, hq, hkv, d, p, rot, seed=case, strided=strided, uniform=uniform)
    k_out = torch.empty((sum(news), hkv, d), dtype=torch.float16, device=dev) if case % 2 else None
    c.check(c.run(lc, inter, k_out=k_out), inter, k_out)
    # the same tokens again at the same places change nothing
    once = [t.clone() for t in (c.k_cache, c.v_cache, c.k_scale, c.v_scale)]
    c.run(lc, inter)
    for a, b in zip(once, (c.k_cache, c.v_cache, c.k_scale, c.v_scale)):
        assert torch.equal(a, b)


def test_append_many_heads_and_tokens_takes_the_chunked_queries(dev):
    """Enough threads for the chip: a thread's angles serve eight heads, the last chunk of them shorter."""
    import langburst_cuda as lc

    print_case("append-chunked")
    for inter in (False, True):
        c = AppendCase(dev, [0], [9000], 61, 1, 256, 64, 128, seed=3)
        c.check(c.run(lc, inter), inter)


def test_append_rotates_in_place_and_without_queries(dev):
    import langburst_cuda as lc
    import torch

    print_case("append-in-place")
    for inter in (False, True):
        c = AppendCase(dev, [9], [50], 4, 2, 128, 16, 64, seed=1, strided=True)
        want = c.run(lc, inter)
        q = c.q.clone()
        lc.kv8_append_out(q, c.k, c.v, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens, c.starts,
                          c.rotation, q, None, inter)
        assert torch.equal(q, want)
        a = AppendCase(dev, [9], [50], 4, 2, 128, 16, 64, seed=1, strided=True)
        lc.kv8_append_out(None, a.k, a.v, a.k_cache, a.v_cache, a.k_scale, a.v_scale, a.table, a.seq_lens, a.starts,
                          a.rotation, None, None, inter)
        for page in (1, 2):  # the pages that hold new tokens alone; which they are is drawn at random
            assert torch.equal(a.k_cache[int(a.table[0, page])], c.k_cache[int(c.table[0, page])])
            assert torch.equal(a.v_scale[int(a.table[0, page])], c.v_scale[int(c.table[0, page])])


def test_append_one_by_one_reaches_the_scales_of_all_at_once(dev):
    """A page filled token by token ends with the scale of the page filled at once, and every value within a step of it."""
    import langburst_cuda as lc
    import torch

    print_case("append-one-by-one")
    d, p, n = 128, 32, 70
    g = _gen(dev, 5)
    x = torch.randn((n, 2, d), device=dev, generator=g).half() * torch.linspace(0.5, 3, n, device=dev)[:, None, None].half()
    pages = torch.arange(3, dtype=torch.int32, device=dev)[None]

    def fresh():
        return (torch.zeros((3, 2, p, d), dtype=torch.int8, device=dev), torch.zeros((3, 2, d, p), dtype=torch.int8, device=dev),
                torch.full((3, 2), 9.0, device=dev), torch.full((3, 2), 9.0, device=dev))

    once, steps = fresh(), fresh()
    lc.kv8_append_out(None, x, x, *once, pages, torch.tensor([n], dtype=torch.int32, device=dev), None, None, None, None)
    for i in range(n):
        lc.kv8_append_out(None, x[i:i + 1], x[i:i + 1], *steps, pages, torch.tensor([i + 1], dtype=torch.int32, device=dev),
                          None, None, None, None)
    torch.cuda.synchronize()
    for a, b in zip(once[2:], steps[2:]):
        assert torch.equal(a, b)
    xs = _np(x)
    for i in range(n):
        step = _np(steps[2][i // p])[:, None]
        # every growth of the scale rounds once more, each by half a step of its time
        assert (np.abs(_np(steps[0][i // p, :, i % p]) * step - xs[i]) <= 6 * step).all()
        assert (np.abs(_np(once[0][i // p, :, i % p]) * step - xs[i]) <= 0.5 * step * (1 + 1e-4)).all()
    assert torch.equal(once[0].transpose(2, 3), once[1]) and torch.equal(steps[0].transpose(2, 3), steps[1])


def test_append_leaves_out_padding_and_missing_pages(dev):
    import langburst_cuda as lc
    import torch

    print_case("append-padding")
    d, p = 64, 16
    c = AppendCase(dev, [0, 10, 20, 30], [4, 4, 4, 4], 2, 1, d, p, 64, seed=2, uniform=True)
    lens = [0, 2, 24, 34]  # no token, the last two of four, and two whole sequences ...
    c.table[2, 1] = -1      # ... one without its page, one with a page number past the cache
    c.table[3, 2] = 10 ** 6
    c.seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = c.run(lc, False)
    assert (q[0:6] == 0).all() and (q[6:] != 0).any()
    rot = _np(c.rotation)
    for t, pos in ((6, 0), (7, 1), (8, 20), (15, 33)):
        want = A.rotate(_np(c.q[t]), rot[pos, :32], rot[pos, 32:], False)
        assert np.abs(_np(q[t]) - want).max() < 0.02
    changed = [i for i in range(c.k_cache.shape[0]) if not torch.equal(c.k_cache[i], c.before[0][i])]
    # of sequence 1 its first page, of sequence 3 its second
    assert set(changed) == {int(c.table[1, 0]), int(c.table[3, 1])}


def test_append_shows_non_finite_values_and_positions_outside_the_table(dev):
    import langburst_cuda as lc
    import torch

    print_case("append-non-finite")
    c = AppendCase(dev, [0, 0], [20, 20], 2, 2, 64, 16, 64, seed=4, positions=18)
    c.k[3, 0, 5], c.v[25, 1, 7] = float("nan"), float("inf")
    q = c.run(lc, False)
    ks, vs = _np(c.k_scale), _np(c.v_scale)
    assert np.isnan(ks[c.table_np[0, 0], 0]) and np.isfinite(ks[c.table_np[0, 0], 1])
    assert np.isinf(vs[c.table_np[1, 0], 1]) and np.isfinite(vs[c.table_np[1, 0], 0])
    assert np.isfinite(_np(q[:18])).all() and np.isnan(_np(q[18:20])).all()
    assert np.isnan(ks[c.table_np[0, 1]]).all()  # its keys have no angle


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_append_to_a_page_with_a_non_finite_scale_keeps_it(dev, bad):
    import langburst_cuda as lc
    import torch

    print_case("append-after-non-finite", bad)
    c = AppendCase(dev, [0, 0], [20, 20], 2, 1, 64, 16, 64, seed=4, positions=32)
    c.k[17, 0, 5], c.v[37, 0, 7] = bad, bad  # the second page of sequence 0, and of sequence 1
    c.run(lc, False)
    table = c.table_np[:, 1]
    for _ in range(2):  # finite tokens after it: what the page held is not known any more, and must not look finite
        c.k[17, 0, 5], c.v[37, 0, 7] = 1.0, 1.0
        lens = c.seq_lens + 1
        rows = torch.tensor([17, 37], device=dev)
        lc.kv8_append_out(None, c.k[rows].contiguous(), c.v[rows].contiguous(), c.k_cache, c.v_cache, c.k_scale, c.v_scale,
                          c.table, lens, None, c.rotation, None, None, False)
        ks, vs = _np(c.k_scale)[table, 0], _np(c.v_scale)[table, 0]
        assert not np.isfinite(ks[0]) and np.isfinite(ks[1]) and np.isfinite(vs[0]) and not np.isfinite(vs[1])


def test_append_of_nothing(dev):
    import langburst_cuda as lc
    import torch

    print_case("append-nothing")
    c = AppendCase(dev, [3, 9], [0, 0], 2, 1, 64, 16, 64)
    c.run(lc, False)
    c.check(torch.empty((0, 2, 64)), False)
    z = AppendCase(dev, [0], [1], 1, 1, 64, 16, 16, uniform=True)  # zeros have scale zero, twice
    z.k.zero_(), z.v.zero_()
    z.run(lc, False)
    cell = z.table_np[0, 0]
    assert float(z.k_scale[cell, 0]) == 0 and float(z.v_scale[cell, 0]) == 0 and not z.k_cache[cell, 0, 0].any()


# --------------------------------------------------------- attention, cache ---

class Cached:
    def __init__(self, dev, lens, n, hq, hkv, d, p, seed=0, scales=None, sharp=1.0):
        import torch

        g = _gen(dev, seed)
        self.lens, self.n, self.hq, self.hkv, self.d, self.p = lens, n, hq, hkv, d, p
        width = max([1] + [-(-x // p) for x in lens]) + 2
        pool = sum(-(-max(x, 0) // p) for x in lens) + 3
        order = torch.randperm(pool - 1).add(1).tolist()  # page 0 is no sequence's
        table = np.full((len(lens), width), 2 ** 30, dtype=np.int32)
        for b, x in enumerate(lens):
            for j in range(-(-max(x, 0) // p)):
                table[b, j] = order.pop()
        self.table_np, self.table = table, torch.from_numpy(table).to(dev)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.k_cache = torch.randint(-127, 128, (pool, hkv, p, d), dtype=torch.int8, device=dev, generator=g)
        self.v_cache = torch.randint(-127, 128, (pool, hkv, d, p), dtype=torch.int8, device=dev, generator=g)
        self.k_scale = torch.rand((pool, hkv), device=dev, generator=g) * 0.02 + 0.002
        self.v_scale = torch.rand((pool, hkv), device=dev, generator=g) * 0.02 + 0.002
        if scales:  # value scales of very different sizes
            self.v_scale *= 10.0 ** torch.randint(-scales, 1, (pool, hkv), device=dev, generator=g)
        free = order + [0]  # what no sequence holds is never used
        self.k_scale[free], self.v_scale[free] = float("nan"), float("inf")
        self.q = (torch.randn((len(lens) * n, hq, d), device=dev, generator=g) * sharp).half()
        self.ws = torch.zeros((max(1, len(lens) * n * hq),), dtype=torch.int32, device=dev)

    def run(self, ops, q=None, out=None, scale=None):
        import torch

        q = self.q if q is None else q
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device=q.device) if out is None else out
        ops.kv8_attention_out(q, self.k_cache, self.v_cache, self.k_scale, self.v_scale, self.table, self.seq_lens, out,
                              self.ws, self.d ** -0.5 if scale is None else scale)
        torch.cuda.synchronize()
        assert not self.ws.any()
        return out

    def keys(self, b, head):
        """The keys and values of the sequence, in 64 bits, and which of them have a page."""
        length, pool = max(self.lens[b], 0), self.k_cache.shape[0]
        pages = self.table_np[b, :-(-length // self.p)]
        has = (pages >= 0) & (pages < pool)
        pages = np.where(has, pages, 0)
        k = _np(self.k_cache[pages, head]) * _np(self.k_scale[pages, head])[:, None, None]
        v = _np(self.v_cache[pages, head]) * _np(self.v_scale[pages, head])[:, None, None]
        k, v = k.reshape(-1, self.d)[:length], v.transpose(0, 2, 1).reshape(-1, self.d)[:length]
        return k, v, np.repeat(has, self.p)[:length]

    def check(self, out, heads=None, scale=None):
        scale = self.d ** -0.5 if scale is None else scale
        got, group = _np(out), self.hq // self.hkv
        for b, length in enumerate(self.lens):
            for h in range(self.hkv) if heads is None else heads:
                k, v, has = self.keys(b, h)
                rows = slice(b * self.n, (b + 1) * self.n)
                for j in range(group):
                    q = _np(self.q[rows, h * group + j])
                    sees = [has[:max(0, length - self.n + i + 1)].sum() for i in range(self.n)]
                    want, spread, _ = A.attend(q, k[has], v[has], scale, sees)
                    w = 2 * A.score_error(q, k[has], scale) + 2.0 ** -18
                    err = np.abs(got[rows, h * group + j] - want)
                    bad = err > 2.0 ** -11 * np.abs(want) + w * spread + 2.0 ** -25
                    assert not bad.any(), (b, h, j, err.max(), np.argwhere(bad)[:3])


CACHED = [
    # lens, n, heads_q, heads_kv, d, page
    ([1], 1, 1, 1, 64, 16),
    ([0, 1, 2, 15, 16, 17], 1, 6, 2, 128, 16),
    ([63, 64, 65, 255, 256, 257], 1, 8, 1, 64, 32),
    ([1000, 0, 3, 511], 1, 24, 4, 256, 64),
    ([2, 3, 700, 40], 3, 10, 2, 128, 32),        # 15 columns, a sequence with fewer tokens than queries
    ([1, 300, 77], 4, 12, 2, 256, 16),           # 24 columns: two blocks of 16
    ([200, 33], 5, 32, 2, 64, 128),              # 80 columns: three blocks of 32
    ([129, 1], 2, 16, 1, 256, 128),              # 32 columns exactly
    ([1] * 70 + [300] + [5] * 70, 1, 2, 2, 64, 16),   # more sequences than a wave has lanes
    ([9000], 1, 6, 1, 128, 16),                  # one long sequence over many workgroups
    ([20000, 30, 5000], 2, 8, 2, 128, 64),       # ragged: parts of three sequences meet in a workgroup
    ([300, 900, 5, 0, 620] * 12, 1, 8, 8, 64, 16),    # about as many pairs as workgroups: most hold a pair
    ([300, 900, 5, 0, 620] * 14, 1, 8, 8, 64, 16),    # and somewhat more pairs than workgroups
    ([9000] + [300] * 31, 1, 8, 4, 128, 32),     # one long sequence among short ones
]


@pytest.mark.parametrize("case", range(len(CACHED)))
def test_attention_over_the_cache_matches_the_definition(dev, case):
    import langburst_cuda as lc
    import torch

    print_case("kv8-attention", case, *CACHED[case][1:])
    c = Cached(dev, *CACHED[case], seed=case)
    out = c.run(lc)
    c.check(out)
    assert torch.equal(out, c.run(lc)), "repeated calls differ"


@pytest.mark.parametrize("sharp,scale", [(0.0, None), (40.0, None), (1.0, 1e-6), (3.0, 1.0)])
def test_attention_over_the_cache_flat_and_sharp_scores(dev, sharp, scale):
    import langburst_cuda as lc

    print_case("kv8-attention-sharp", sharp, scale)
    c = Cached(dev, [777, 20], 2, 4, 2, 128, 32, seed=1, sharp=sharp)
    c.check(c.run(lc, scale=scale), scale=scale)


@pytest.mark.parametrize("d,hkv", [(64, 4), (128, 2), (256, 1)])
def test_attention_over_the_cache_rounds_its_weights_once(dev, d, hkv):
    """Thousands of rows with few keys, so that a single weight rounded twice shows: outputs are within a rounding of exact."""
    import langburst_cuda as lc

    print_case("kv8-attention-weights", d, hkv)
    for seed in range(12):
        c = Cached(dev, [9 + 8 * i for i in range(8)], 1, 8 * hkv, hkv, d, 16, seed=100 + seed)
        c.check(c.run(lc))


@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (8, 2, 128), (6, 1, 256)])
def test_attention_over_the_cache_with_cold_caches(dev, hq, hkv, d):
    """One step of tokens a workgroup, and nothing of them in the GPU's caches: the loads take their longest."""
    import langburst_cuda as lc
    import torch

    print_case("kv8-attention-cold", hq, hkv, d)
    c = Cached(dev, [40, 256, 7000], 1, hq, hkv, d, 64, seed=4)
    c.check(c.run(lc))
    want = c.run(lc)
    flush = torch.empty(2 ** 29, dtype=torch.uint8, device=dev)
    for i in range(20):
        flush.fill_(i)
        assert torch.equal(c.run(lc), want), i


def test_attention_over_pages_of_very_different_scales(dev):
    import langburst_cuda as lc

    print_case("kv8-attention-scales")
    c = Cached(dev, [900, 40], 1, 4, 2, 64, 16, seed=2, scales=6)
    c.v_scale[int(c.table[0, 3])] = 0  # a page of zeros counts in the softmax
    out = c.run(lc)
    c.check(out)


def test_attention_skips_tokens_without_a_page(dev):
    import langburst_cuda as lc

    print_case("kv8-attention-missing")
    c = Cached(dev, [300, 100, 40], 1, 4, 2, 128, 32, seed=3)
    c.table_np[0, 2], c.table_np[0, 9], c.table_np[1, :] = -1, 10 ** 6, -1
    c.table.copy_(c.table.new_tensor(c.table_np))
    out = c.run(lc)
    c.check(out)
    assert (out[1] == 0).all()


def test_attention_of_strided_rows_other_streams_and_longer_lengths(dev):
    import langburst_cuda as lc
    import torch

    print_case("kv8-attention-strided")
    c = Cached(dev, [300, 64], 2, 6, 2, 128, 16, seed=4)
    want = c.run(lc)
    wide = torch.zeros((4, 7, 256), dtype=torch.float16, device=dev)
    wide[:, 1:, :128] = c.q
    out = torch.full((4, 9, 256), 7.0, dtype=torch.float16, device=dev)
    assert torch.equal(c.run(lc, q=wide[:, 1:, :128], out=out[:, 2:8, 128:]), want)
    assert (out[:, :2] == 7).all() and (out[:, 8:] == 7).all() and (out[:, :, :128] == 7).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(c.run(lc), want)
    # a length past the table is the table's
    c = Cached(dev, [18 * 16], 1, 2, 1, 64, 16, seed=5)
    c.table = c.table[:, :18].contiguous()
    want = c.run(lc)
    c.seq_lens.fill_(10 ** 6)
    assert torch.equal(c.run(lc), want)


def test_attention_cache_larger_than_32_bit_offsets(dev):
    import langburst_cuda as lc
    import torch

    p, hkv, d = 128, 4, 256
    pool = (1 << 32) // (p * hkv * d) + 40
    print_case("kv8-attention-4GiB", pool)
    small = Cached(dev, [500], 1, 8, hkv, d, p, seed=6)
    want = small.run(lc)
    k = torch.empty((pool, hkv, p, d), dtype=torch.int8, device=dev)
    v = torch.empty((pool, hkv, d, p), dtype=torch.int8, device=dev)
    ks, vs = torch.zeros((pool, hkv), device=dev), torch.zeros((pool, hkv), device=dev)
    pages = torch.tensor([pool - 1, pool - 30, 1, pool - 7], device=dev)
    old = small.table[0, :4].long()
    k[pages], v[pages], ks[pages], vs[pages] = small.k_cache[old], small.v_cache[old], small.k_scale[old], small.v_scale[old]
    small.k_cache, small.v_cache, small.k_scale, small.v_scale = k, v, ks, vs
    small.table = pages.to(torch.int32)[None].contiguous()
    assert torch.equal(small.run(lc), want)
    # and the writer reaches the same places
    x = torch.randn((500, hkv, d), device=dev).half()
    lens = torch.tensor([500], dtype=torch.int32, device=dev)
    lc.kv8_append_out(None, x, x, k, v, ks, vs, small.table, lens, None, None, None, None)
    torch.cuda.synchronize()
    got = _np(k[pages].transpose(1, 2).reshape(-1, hkv, d)[:500]) * np.repeat(_np(ks[pages]), p, 0)[:500, :, None]
    assert (np.abs(got - _np(x)) <= 0.51 * np.repeat(_np(ks[pages]), p, 0)[:500, :, None]).all()


# ----------------------------------------------------------------- prompts ---

def _prompt(dev, lens, hq, hkv, d, seed=0, strided=False, extra=0):
    import torch

    g = _gen(dev, seed)
    t = sum(lens) + extra
    if strided:
        x = torch.randn((t, hq + 2 * hkv + 1, 2 * d), device=dev, generator=g).half()[:, 1:, d:]
    else:
        x = torch.randn((t, hq + 2 * hkv, d), device=dev, generator=g).half()
    starts = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=dev)
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], starts


def _check_prompt(out, q, k, v, lens, scale, heads=None, rows=None):
    hq, hkv = q.shape[1], k.shape[1]
    at = 0
    for n in lens:
        for h in range(hq) if heads is None else heads:
            kk, vv = _np(k[at:at + n, h // (hq // hkv)]), _np(v[at:at + n, h // (hq // hkv)])
            pick = np.arange(n) if rows is None else np.unique(np.clip(rows, 0, max(n - 1, 0)))[:n]
            qq = _np(q[at:at + n, h])[pick]
            want, spread, total = A.attend(qq, kk, vv, scale, pick + 1)
            w = 2 * A.score_error(qq, kk, scale) + 2.0 ** -18 + 2.0 ** -11
            err = np.abs(_np(out[at:at + n, h])[pick] - want)
            bad = err > 2.0 ** -11 * np.abs(want) + w * spread + 2.0 ** -32 * total + 2.0 ** -25
            assert not bad.any(), (n, h, err.max(), pick[np.argwhere(bad)[:3, 0]])
        at += n


PROMPTS = [
    # lens, heads_q, heads_kv, d
    ([1], 1, 1, 64),
    ([1, 2, 0, 63, 64, 65], 4, 2, 128),
    ([127, 128, 129], 3, 3, 64),
    ([300, 1, 0, 0, 257], 6, 1, 256),
    ([511], 10, 2, 128),
    ([97, 210], 16, 1, 256),
    ([33] * 66 + [7] * 66, 2, 1, 64),            # more sequences than a wave has lanes
    ([40, 500], 7, 1, 128),
    ([260, 5], 64, 1, 64),
]


@pytest.mark.parametrize("case", range(len(PROMPTS)))
@pytest.mark.parametrize("strided", [False, True])
def test_prompt_attention_matches_the_definition(dev, case, strided):
    import langburst_cuda as lc
    import torch

    lens, hq, hkv, d = PROMPTS[case]
    print_case("prompt", case, strided)
    q, k, v, starts = _prompt(dev, lens, hq, hkv, d, seed=case, strided=strided, extra=5)
    out = torch.full((sum(lens) + 5, hq, d), 7.0, dtype=torch.float16, device=dev)
    lc.prompt_attention_out(q, k, v, starts, out, d ** -0.5)
    torch.cuda.synchronize()
    _check_prompt(out, q, k, v, lens, d ** -0.5)
    assert (out[sum(lens):] == 7).all()
    again = torch.empty_like(out).fill_(7.0)
    lc.prompt_attention_out(q, k, v, starts, again, d ** -0.5)
    assert torch.equal(out, again)


@pytest.mark.parametrize("hq,hkv,d,n", [(40, 8, 128, 2100), (24, 4, 256, 1300), (4, 4, 64, 4001)])
def test_prompt_attention_long(dev, hq, hkv, d, n):
    import langburst_cuda as lc
    import torch

    print_case("prompt-long", hq, hkv, d, n)
    q, k, v, _ = _prompt(dev, [n], hq, hkv, d, seed=n)
    out = torch.empty((n, hq, d), dtype=torch.float16, device=dev)
    lc.prompt_attention_out(q, k, v, None, out, d ** -0.5)
    torch.cuda.synchronize()
    rows = np.unique(np.concatenate([np.arange(0, n, 61), np.arange(n - 70, n), np.arange(130)]))
    _check_prompt(out, q, k, v, [n], d ** -0.5, heads=(0, hq // 2, hq - 1), rows=rows)


@pytest.mark.parametrize("factor,scale", [(0.0, None), (30.0, None), (1.0, 1e-6), (3.0, 1.0)])
def test_prompt_attention_flat_and_sharp_scores(dev, factor, scale):
    import langburst_cuda as lc
    import torch

    print_case("prompt-sharp", factor, scale)
    q, k, v, starts = _prompt(dev, [400, 70], 4, 2, 128, seed=1)
    q, scale = q * factor, scale or 128 ** -0.5
    out = torch.empty((470, 4, 128), dtype=torch.float16, device=dev)
    lc.prompt_attention_out(q, k, v, starts, out, scale)
    torch.cuda.synchronize()
    _check_prompt(out, q, k, v, [400, 70], scale)


def test_prompt_attention_keeps_sequences_apart(dev):
    """What is not finite in one sequence, or after the last, reaches no other."""
    import langburst_cuda as lc
    import torch

    print_case("prompt-apart")
    for d in (64, 128, 256):
        lens = [70, 10, 130]
        q, k, v, starts = _prompt(dev, lens, 4, 2, d, seed=d, extra=50)
        want = torch.zeros((260, 4, d), dtype=torch.float16, device=dev)
        lc.prompt_attention_out(q, k, v, starts, want, d ** -0.5)
        for x in (q, k, v):
            x[70:80], x[210:] = float("nan"), float("inf")
        out = torch.zeros_like(want)
        lc.prompt_attention_out(q, k, v, starts, out, d ** -0.5)
        torch.cuda.synchronize()
        keep = list(range(70)) + list(range(80, 210))
        assert torch.equal(out[keep], want[keep]) and torch.isnan(out[70:80]).all() and not out[210:].any()


# --------------------------------------------------- graphs and the wrappers ---

@pytest.mark.parametrize("own", [False, True])
def test_cache_attend_captured_before_its_first_eager_call(dev, own):
    """A workspace made in a capture is zeroed by replays alone: no eager call may take it."""
    import torch

    from neurova_amd.attention import KV8Cache

    print_case("attend-captured-first", own)
    c = Cached(dev, [2000, 77, 600], 1, 8, 2, 128, 32, seed=6)
    cache = KV8Cache(*c.k_cache.shape[:2], 128, page_size=32, device=dev)
    cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale = c.k_cache, c.v_cache, c.k_scale, c.v_scale
    ws = torch.zeros(c.q.shape[0] * c.q.shape[1], dtype=torch.int32, device=dev) if own else None
    out = torch.empty_like(c.q)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            cache.attend(c.q, c.table, c.seq_lens, out=out, workspace=ws)
        assert not cache._workspaces
        c.check(cache.attend(c.q, c.table, c.seq_lens))
        eager = cache.attend(c.q, c.table, c.seq_lens)
    torch.cuda.synchronize()
    for _ in range(4):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        with torch.cuda.stream(side):
            assert torch.equal(cache.attend(c.q, c.table, c.seq_lens), eager)
        torch.cuda.synchronize()


def test_operators_replay_from_graphs(dev):
    """Each operator captured, replayed with eager work between, equal to its eager result every time."""
    import langburst_cuda as lc
    import torch

    print_case("attention-graphs")
    c = Cached(dev, [5000, 300, 0], 2, 8, 2, 128, 64, seed=8)
    a = AppendCase(dev, [40, 0], [1, 1], 8, 2, 128, 64, 128, seed=9, uniform=True)
    q, k, v, starts = _prompt(dev, [300, 20], 8, 2, 128, seed=10)
    want_c, want_a = c.run(lc), a.run(lc, False)
    want_p = torch.empty(q.shape, dtype=torch.float16, device=dev)
    lc.prompt_attention_out(q, k, v, starts, want_p, 0.1)
    caches = [t.clone() for t in (a.k_cache, a.v_cache, a.k_scale, a.v_scale)]
    out_c, out_a, out_p = torch.empty_like(want_c), torch.empty_like(want_a), torch.empty_like(want_p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            lc.kv8_append_out(a.q, a.k, a.v, a.k_cache, a.v_cache, a.k_scale, a.v_scale, a.table, a.seq_lens, None,
                              a.rotation, out_a, None, False)
            lc.kv8_attention_out(c.q, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens, out_c, c.ws, c.d ** -0.5)
            lc.prompt_attention_out(q, k, v, starts, out_p, 0.1)
    torch.cuda.synchronize()
    for _ in range(4):
        for o in (out_c, out_a, out_p):
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_c, want_c) and torch.equal(out_a, want_a) and torch.equal(out_p, want_p)
        for x, y in zip(caches, (a.k_cache, a.v_cache, a.k_scale, a.v_scale)):
            assert torch.equal(x, y)
        assert not c.ws.any()
        Cached(dev, [700], 1, 8, 2, 128, 64, seed=11).run(lc)  # eager work between the replays


def test_c_abi_calls_match_the_module(dev):
    import torch

    import langburst_cuda as lc
    from neurova_amd import capi

    print_case("attention-capi")
    c = Cached(dev, [600, 9], 2, 6, 2, 128, 32, seed=12)
    want = c.run(lc)
    nbytes = capi.kv8_attention_scratch_bytes(2, 4, 6, 2, 128, 32, c.table.shape[1])
    scratch = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    out = torch.empty_like(want)
    assert capi.kv8_attention(c.q, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens, out, c.ws, scratch,
                              128 ** -0.5) == capi.LB_OK
    assert torch.equal(out, want)
    assert capi.kv8_attention(c.q, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens, out, c.ws,
                              scratch[:16], 128 ** -0.5) == capi.LB_ERR_SCRATCH
    assert capi.kv8_attention(c.q, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens, out, c.ws[:3],
                              scratch, 128 ** -0.5) == capi.LB_ERR_WORKSPACE
    a, b = (AppendCase(dev, [40], [30], 4, 2, 64, 16, 64, seed=13) for _ in range(2))
    want = a.run(lc, True)
    out = torch.empty_like(want)
    assert capi.kv8_append(b.q, b.k, b.v, b.k_cache, b.v_cache, b.k_scale, b.v_scale, b.table, b.seq_lens, b.starts,
                           b.rotation, out, None, True) == capi.LB_OK
    assert torch.equal(out, want)
    q, k, v, starts = _prompt(dev, [100, 30], 4, 2, 64, seed=14)
    want, out = torch.empty((130, 4, 64), dtype=torch.float16, device=dev), torch.empty((130, 4, 64), dtype=torch.float16, device=dev)
    lc.prompt_attention_out(q, k, v, starts, want, 0.125)
    assert capi.prompt_attention(q, k, v, starts, out, 0.125) == capi.LB_OK
    assert torch.equal(out, want)


def test_refusals_of_the_module(dev):
    import langburst_cuda as lc
    import torch

    print_case("attention-refusals")
    c = Cached(dev, [30], 1, 4, 2, 64, 16)

    def attend(**kw):
        a = dict(q=c.q, k_cache=c.k_cache, v_cache=c.v_cache, k_scale=c.k_scale, v_scale=c.v_scale, page_table=c.table,
                 seq_lens=c.seq_lens, out=torch.empty_like(c.q), workspace=c.ws, softmax_scale=0.125)
        a.update(kw)
        lc.kv8_attention_out(**a)

    attend()
    for kw, text in [(dict(q=c.q.float()), "q must be fp16"), (dict(q=c.q[:, :3]), "heads_q must be a multiple"),
                     (dict(v_cache=c.k_cache), "v_cache must be"), (dict(k_scale=c.k_scale.half()), "k_scale must be fp32"),
                     (dict(page_table=c.table.long()), "page_table must be int32"), (dict(softmax_scale=0.0), "softmax_scale"),
                     (dict(seq_lens=c.seq_lens.cpu()), "must be CUDA"), (dict(out=torch.empty_like(c.q)[:, :2]), "out must have q's shape"),
                     (dict(workspace=c.ws[:0]), "workspace too small"), (dict(q=c.q[..., 1:]), "q must"),
                     (dict(seq_lens=c.seq_lens.repeat(2)), "page_table must be"), (dict(softmax_scale=float("nan")), "softmax_scale")]:
        with pytest.raises(RuntimeError, match=text):
            attend(**kw)
    a = AppendCase(dev, [0], [8], 4, 2, 64, 16, 64)

    def append(**kw):
        d = dict(q=a.q, k=a.k, v=a.v, k_cache=a.k_cache, v_cache=a.v_cache, k_scale=a.k_scale, v_scale=a.v_scale,
                 page_table=a.table, seq_lens=a.seq_lens, cu_seqlens=a.starts, cos_sin=a.rotation,
                 q_out=torch.empty_like(a.q), k_out=None)
        d.update(kw)
        lc.kv8_append_out(**d)

    append()
    for kw, text in [(dict(q_out=None), "given together"), (dict(k=a.k[:, :1]), "k must be"), (dict(v=a.v[:4]), "v must have"),
                     (dict(k_out=a.k), "k_out must not be k"), (dict(cos_sin=a.rotation[:, :24].contiguous()), "rot_dim"),
                     (dict(cos_sin=a.rotation[:, :32]), "cos_sin must be contiguous"), (dict(cu_seqlens=a.starts[:1]), "cu_seqlens must be"),
                     (dict(cu_seqlens=None, seq_lens=a.seq_lens.repeat(3), page_table=a.table.repeat(3, 1)), "same number of tokens"),
                     (dict(k=a.k.to(torch.bfloat16)), "k must be fp16")]:
        with pytest.raises(RuntimeError, match=text):
            append(**kw)
    q, k, v, starts = _prompt(dev, [20], 4, 2, 64)
    for args, text in [((q[:, :3], k, v, starts, q[:, :3]), "heads_q must be a multiple"), ((q, k, v[:10], starts, q), "v must have"),
                       ((q, k, v, starts.long(), q), "int32"), ((q[..., :32], k[..., :32], v[..., :32], starts, q), "head_dim must be"),
                       ((q, k, v, starts, q[:5]), "out must have"), ((q.transpose(1, 2), k, v, starts, q), "contiguous along head_dim")]:
        with pytest.raises(RuntimeError, match=text):
            lc.prompt_attention_out(*args, 0.125)


def test_layer_between_projections(dev):
    """A prompt, then tokens one by one, through the cache object: decoding agrees with the prompt's attention over the same tokens."""
    import torch

    from neurova_amd.attention import KV8Cache, prompt_attention, rotation_table

    print_case("attention-layer")
    hq, hkv, d, n, more = 6, 2, 128, 90, 5
    g = _gen(dev, 21)
    qkv = torch.randn((n + more, hq + 2 * hkv, d), device=dev, generator=g).half()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    table = rotation_table(n + more, 64, scaling="yarn", factor=4, original_positions=32, device=dev)
    cache = KV8Cache(8, hkv, d, page_size=32, device=dev)
    pages = torch.tensor([[5, 2, 7]], dtype=torch.int32, device=dev)

    def lens(x):
        return torch.tensor([x], dtype=torch.int32, device=dev)

    whole = KV8Cache(8, hkv, d, page_size=32, device=dev)
    qr, kr = whole.append(q, k, v, pages, lens(n + more), rotation=table, return_k=True)
    want = prompt_attention(qr, kr, v)
    cache.append(q[:n], k[:n], v[:n], pages, lens(n), torch.tensor([0, n], dtype=torch.int32, device=dev), rotation=table)
    for i in range(n, n + more):
        row = q[i:i + 1].clone()
        cache.append(row, k[i:i + 1], v[i:i + 1], pages, lens(i + 1), rotation=table, q_out=row)
        assert torch.equal(row, qr[i:i + 1])
        got = cache.attend(row, pages, lens(i + 1))
        # 8-bit values: a step is max / 127 of about three, a value's error uniform in half a step, and the output an
        # average of them; the keys' errors move scores of about one by as much
        assert (got - want[i:i + 1]).abs().max() < 0.05
