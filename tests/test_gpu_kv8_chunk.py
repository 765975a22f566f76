"""Attention of packed chunks of new tokens over the 8-bit pages, against the definition in 64 bits.

Tolerance of an output, set before any run: its rounding 2^-11 |o|, the error
of the weights times sum p |v|, and 2^-25 for subnormals.  A weight's error is
twice that of its score in fp32 (numerator and denominator), the hardware's
exponential, logarithm and sums (2^-17) and its rounding to fp16 (2^-11); one
below fp16's normal numbers is off by 2^-32 of the row's largest weight times
value scale.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests.gpu_util import print_case

pytestmark = pytest.mark.gpu


def attend64(q, codes_k, ks, codes_v, vs, scale, sees):
    """q [n, d], codes [m, d], scales [m], sees bool [n, m], all in 64 bits: the output and its tolerance."""
    import torch

    k = codes_k * ks[:, None]
    s = ((q @ k.T) * scale).masked_fill(~sees, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -torch.inf, 0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1)
    w = p * vs
    out, spread = w @ codes_v, w.abs() @ codes_v.abs()
    score = (q.shape[1] + 3) * 2.0 ** -24 * float((q.abs() @ k.abs().T).max()) * scale
    tiny = 2.0 ** -32 * w.abs().amax(-1, keepdim=True) * (sees.double() @ codes_v.abs())
    return out, 2.0 ** -11 * out.abs() + (2 * score + 2.0 ** -17 + 2.0 ** -11) * spread + tiny + 2.0 ** -25


class Chunks:
    """`news` tokens of every sequence after `held` ones (less than none: padding first), over pages in random order."""

    def __init__(self, dev, news, held, hq, hkv, d, p, seed=0, sharp=1.0, spread=0.0, extra=0, wide=2):
        import torch

        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        self.dev, self.news, self.hq, self.hkv, self.d, self.p = dev, news, hq, hkv, d, p
        self.lens = [max(n + h, 0) for n, h in zip(news, held)]
        counts = [-(-x // p) for x in self.lens]
        pool, width = sum(counts) + 3, max(counts + [0]) + wide
        order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table_np = np.full((len(news), width), -5, dtype=np.int32)
        for b, c in enumerate(counts):
            for j in range(c):
                self.table_np[b, j] = order.pop()
        self.table = torch.from_numpy(self.table_np.copy()).to(dev)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        self.starts = torch.tensor(np.cumsum([0] + news), dtype=torch.int32, device=dev)
        self.q = (torch.randn((sum(news) + extra, hq, d), device=dev, generator=g) * sharp).half()
        self.k_cache = torch.randint(-127, 128, (pool, hkv, p, d), dtype=torch.int8, device=dev, generator=g)
        self.v_cache = torch.randint(-127, 128, (pool, hkv, d, p), dtype=torch.int8, device=dev, generator=g)
        self.k_scale, self.v_scale = ((torch.randn((pool, hkv), device=dev, generator=g) * spread).exp2() *
                                      (torch.rand((pool, hkv), device=dev, generator=g) * 0.015 + 0.005) for _ in range(2))

    def run(self, q=None, out=None, scale=None):
        import langburst_cuda as lc
        import torch

        q = self.q if q is None else q
        out = torch.full(q.shape, 7.0, dtype=torch.float16, device=self.dev) if out is None else out
        lc.kv8_chunk_attention_out(q, self.k_cache, self.v_cache, self.k_scale, self.v_scale, self.table, self.seq_lens, self.starts,
                                   out, self.d ** -0.5 if scale is None else scale)
        return out

    def check(self, out, heads=None, scale=None, most=None):
        """`most`: at most this many rows of a sequence are looked at, the first and the last among them."""
        import torch

        scale, at, pool = self.d ** -0.5 if scale is None else scale, 0, self.k_cache.shape[0]
        for b, (n, length) in enumerate(zip(self.news, self.lens)):
            rows = np.arange(n)
            if most and n > most:
                rows = np.unique(np.concatenate([rows[:most // 3], rows[-(most // 3):], rows[::max(1, 3 * n // most)]]))
            kept = min(length, self.table.shape[1] * self.p)
            pages = torch.from_numpy(self.table_np[b, :-(-kept // self.p)]).to(self.dev).long()
            has = (pages >= 0) & (pages < pool)
            pages = pages.where(has, 0)
            sees = torch.from_numpy(length - n + rows).to(self.dev)[:, None] >= torch.arange(kept, device=self.dev)
            sees &= has.repeat_interleave(self.p)[:kept]
            for h in range(self.hq) if heads is None else heads:
                g = h // (self.hq // self.hkv)
                ck = self.k_cache[pages, g].double().reshape(-1, self.d)[:kept]
                cv = self.v_cache[pages, g].double().transpose(1, 2).reshape(-1, self.d)[:kept]
                ks, vs = (t[pages, g].double().repeat_interleave(self.p)[:kept] for t in (self.k_scale, self.v_scale))
                where = at + torch.from_numpy(rows).to(self.dev)
                got = out[where, h].double()
                if kept == 0 or n == 0:
                    assert not got.any(), (b, h)
                    continue
                want, bound = attend64(self.q[where, h].double(), ck, ks, cv, vs, scale, sees)
                bad = ~((got - want).abs() <= bound)
                assert not bad.any(), (b, h, float((got - want).abs().max()), bad.nonzero()[:3].tolist(), int(bad.sum()))
            at += n
        assert (out[at:] == 7).all()


CHUNKS = [
    # new tokens, tokens held before, heads_q, heads_kv, d, page
    ([1], [0], 1, 1, 64, 16),
    ([1, 2, 3, 0, 17], [0, 0, 13, 40, 47], 2, 1, 128, 16),
    ([64, 63, 65], [0, 1, 63], 4, 2, 64, 32),
    ([24], [301], 24, 4, 256, 64),
    ([130, 1, 5], [0, 700, 250], 10, 2, 128, 128),
    ([40, 3], [-7, -3], 6, 2, 128, 16),               # padding before position 0; a sequence of padding alone
    ([200, 33], [1, 500], 3, 3, 256, 16),
    ([77], [2000], 16, 1, 64, 128),
    ([50, 1, 1, 90], [3000, 4000, 10, 0], 5, 1, 128, 32),   # cut keys beside whole ones
    ([1] * 70 + [150] + [2] * 9, [5] * 30 + [300] * 50, 2, 2, 64, 16),   # more sequences than a wave has lanes
    ([9], [9000], 7, 1, 256, 32),                     # few rows over many workgroups
    ([129, 260], [1500, 100], 12, 1, 256, 64),
    ([31, 600], [50, 33], 8, 8, 64, 16),
    ([4] * 20, [100, 900, 40, 2000] * 5, 20, 4, 128, 16),
    # more pieces than run at once: the sequences with the longest come first, whatever their place
    ([1, 2, 1] * 34, [20, 300, 70, 5, 150, 0] * 17, 8, 8, 64, 32),
    ([1, 0, 3, 1] * 65, [20, 0, 300, 70] * 65, 3, 3, 64, 16),      # and more sequences than stay in registers
    ([40] * 12, [300, 100, 200] * 4, 64, 8, 64, 16),
]


@pytest.mark.parametrize("case", range(len(CHUNKS)))
def test_chunks_match_the_definition(dev, case):
    import torch

    print_case("chunk", case, *CHUNKS[case][2:])
    c = Chunks(dev, *CHUNKS[case], seed=case, extra=3)
    out = c.run()
    torch.cuda.synchronize()
    c.check(out)
    assert torch.equal(out, c.run()), "repeated calls differ"


@pytest.mark.parametrize("news,held,hq,hkv,d,p", [([1500], [700], 40, 8, 128, 16), ([600, 1, 300], [0, 9000, 1000], 24, 4, 256, 64),
                                                   ([2500, 70], [0, 4000], 8, 8, 64, 32), ([3], [40000], 8, 2, 128, 64),
                                                   # whole row blocks for a round, and the first ones cut so that they fill one more
                                                   ([1100], [300], 64, 2, 256, 32), ([2300], [900], 32, 4, 128, 16), ([2300], [0], 32, 4, 64, 64)])
def test_long_chunks(dev, news, held, hq, hkv, d, p):
    import torch

    print_case("chunk-long", news, held, hq, hkv, d, p)
    c = Chunks(dev, news, held, hq, hkv, d, p, seed=d)
    out = c.run()
    torch.cuda.synchronize()
    c.check(out, heads=(0, hq // 2, hq - 1), most=90)


@pytest.mark.parametrize("sharp,scale", [(0.0, None), (20.0, None), (1.0, 1e-6), (3.0, 1.0)])
def test_flat_and_sharp_scores(dev, sharp, scale):
    print_case("chunk-sharp", sharp, scale)
    for d in (64, 128, 256):
        c = Chunks(dev, [90, 3], [300, 70], 4, 2, d, 32, seed=1, sharp=sharp)
        c.check(c.run(scale=scale), scale=scale)


@pytest.mark.parametrize("spread", [3.0, 9.0])
def test_pages_of_very_different_scales(dev, spread):
    """Scales of either kind spread over their logarithm, so far that tiles leave the range of the common way; a page of zeros counts in the softmax."""
    print_case("chunk-scales", spread)
    for d, p in ((64, 16), (128, 64), (256, 32)):
        c = Chunks(dev, [70, 5], [500, 90], 4, 2, d, p, seed=2, spread=spread, sharp=2.0 ** -spread)
        c.v_scale[int(c.table[0, 3])] = 0
        c.k_scale[int(c.table[0, 1])] = 0
        c.check(c.run())


def test_negative_scales_and_values_near_the_ends_of_fp32(dev):
    print_case("chunk-negative")
    c = Chunks(dev, [70, 5], [500, 90], 4, 2, 128, 16, seed=3)
    c.k_scale[::3] *= -1
    c.v_scale[::2] *= -1
    c.check(c.run())
    c = Chunks(dev, [40], [200], 2, 1, 64, 16, seed=4)
    c.v_scale[int(c.table[0, 2])] = 2.0 ** -79
    c.v_scale[int(c.table[0, 5])] = 1e-45  # subnormal: its values count as zeros
    got = c.run()
    c.v_scale[int(c.table[0, 5])] = 0
    c.check(got)


def test_tokens_without_a_page_are_not_seen(dev):
    import torch

    print_case("chunk-missing")
    for d, p in ((64, 16), (128, 32), (256, 128)):
        c = Chunks(dev, [60, 20, 9], [300, 100, 40], 4, 2, d, p, seed=3)
        c.table_np[0, 0], c.table_np[0, 2], c.table_np[1, :] = -1, 10 ** 6, -1
        c.table.copy_(torch.from_numpy(c.table_np))
        out = c.run()
        c.check(out)
        assert (out[60:80] == 0).all()


def test_lengths_past_the_table_and_below_zero(dev):
    import torch

    print_case("chunk-past")
    c = Chunks(dev, [50, 8], [250, 100], 2, 1, 128, 16, seed=5, wide=0)
    c.lens[0] += 40  # past the table's 300 and some tokens: rows see up to their own of what the table holds
    c.seq_lens[0] += 40
    c.check(c.run())
    c.lens[0] = 10 ** 6
    c.seq_lens[0] = 10 ** 6
    c.check(c.run())
    c.seq_lens.copy_(torch.tensor([-4, -2 ** 31], dtype=torch.int32))
    assert not c.run().any()


@pytest.mark.parametrize("kind", ["k_scale", "v_scale"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_scale_that_is_not_finite_reaches_the_rows_that_see_its_page(dev, kind, value):
    import torch

    print_case("chunk-non-finite", kind, value)
    for d, p in ((64, 16), (128, 32), (256, 64)):
        c = Chunks(dev, [150, 40], [30, 90], 4, 2, d, p, seed=6)
        want = c.run()
        page = 96 // p  # of the first sequence: positions 96 and on, seen from its row 66 on
        getattr(c, kind)[int(c.table[0, page]), 1] = value
        out = c.run()
        torch.cuda.synchronize()
        first = page * p - 30
        assert torch.equal(out[:, :2], want[:, :2])          # the other head
        assert torch.equal(out[:first], want[:first]) and torch.equal(out[150:], want[150:])
        assert (~torch.isfinite(out[first:150, 2:])).any(-1).all()


def test_what_follows_a_sequence_in_its_last_page_is_not_read(dev):
    """Codes behind the last token, and pages of the table behind it, change nothing."""
    import torch

    print_case("chunk-behind")
    c = Chunks(dev, [20, 33], [25, 100], 4, 2, 128, 64, seed=7)
    want = c.run()
    for b, n in enumerate(c.lens):
        last = int(c.table_np[b, n // 64])
        c.k_cache[last, :, n % 64:] = 127
        c.v_cache[last, :, :, n % 64:] = -127
        c.table[b, n // 64 + 1:] = 10 ** 9
    assert torch.equal(c.run(), want)


def test_strided_rows_other_streams_and_shared_pages(dev):
    import torch

    print_case("chunk-strided")
    c = Chunks(dev, [30, 64], [300, 20], 6, 2, 128, 16, seed=8)
    want = c.run()
    wide = torch.zeros((94, 7, 256), dtype=torch.float16, device=dev)
    wide[:, 1:, :128] = c.q
    out = torch.full((94, 9, 256), 7.0, dtype=torch.float16, device=dev)
    assert torch.equal(c.run(q=wide[:, 1:, :128], out=out[:, 2:8, 128:]), want)
    assert (out[:, :2] == 7).all() and (out[:, 8:] == 7).all() and (out[:, :, :128] == 7).all()
    rows = torch.full((6, 94, 128), 7.0, dtype=torch.float16, device=dev).transpose(0, 1)   # heads outside tokens
    assert torch.equal(c.run(out=rows), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(c.run(), want)
    torch.cuda.current_stream().wait_stream(side)
    # both sequences over the pages of the first, and a table whose rows lie apart
    apart = torch.full((2, c.table.shape[1] + 5), -1, dtype=torch.int32, device=dev)[:, 2:-3]
    apart[:] = c.table[0]
    c.table, c.table_np[1] = apart, c.table_np[0]
    c.check(c.run())


def test_packed_starts_that_leave_tokens_out(dev):
    """Tokens before the first sequence, between two and after the last stay as they are; starts outside the rows are cut to them."""
    import torch

    print_case("chunk-starts")
    c = Chunks(dev, [10, 20], [40, 200], 4, 2, 64, 16, seed=9)
    want = c.run()
    c.q = torch.cat([c.q[:5], c.q, c.q[:9]])
    c.starts = torch.tensor([5, 15, 35], dtype=torch.int32, device=dev)
    out = c.run()
    assert torch.equal(out[5:35], want) and (out[:5] == 7).all() and (out[35:] == 7).all()
    c.starts = torch.tensor([-3, 15, 10 ** 6], dtype=torch.int32, device=dev)
    out = c.run()
    assert (out != 7).any(-1).all()
    c.starts = torch.tensor([30, 10, 5], dtype=torch.int32, device=dev)
    assert (c.run() == 7).all()


def test_a_cache_larger_than_32_bit_offsets(dev):
    import torch

    p, hkv, d = 128, 4, 256
    pool = (1 << 32) // (p * hkv * d) + 40
    print_case("chunk-4GiB", pool)
    c = Chunks(dev, [70], [430], 8, hkv, d, p, seed=10)
    want = c.run()
    pages = torch.tensor([pool - 1, pool - 30, 1, pool - 7], device=dev)
    old = c.table[0, :4].long()
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        t = getattr(c, name)
        big = torch.empty((pool, *t.shape[1:]), dtype=t.dtype, device=dev)
        big[pages] = t[old]
        setattr(c, name, big)
    c.table = pages.to(torch.int32)[None].contiguous()
    assert torch.equal(c.run(), want)


def test_chunks_captured_into_graphs(dev):
    """Two graphs of different sizes, lengths that change between their replays, and eager calls between."""
    import torch

    print_case("chunk-graphs")
    a, b = Chunks(dev, [40, 1, 1], [3000, 700, 2], 8, 2, 128, 16, seed=11), Chunks(dev, [200], [900], 6, 1, 256, 64, seed=12)
    outs = [torch.empty_like(a.q), torch.empty_like(b.q)]
    graphs, side = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for c, o, graph in zip((a, b), outs, graphs):
            with torch.cuda.graph(graph, stream=side):
                c.run(out=o)
    torch.cuda.synchronize()
    for i in range(4):
        a.lens = [3040 - 700 * i, 701, 3]
        a.seq_lens.copy_(torch.tensor(a.lens, dtype=torch.int32))
        for c, o, graph in zip((a, b), outs, graphs):
            o.fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        for c, o in zip((a, b), outs):
            assert torch.equal(o, c.run()), i
        a.check(outs[0])


def test_chunks_through_the_cache_and_the_c_abi(dev):
    """Prompts that arrive in pieces see what they would see at once, and decode beside other pieces."""
    import torch

    from neurova_amd import capi
    from neurova_amd.attention import KV8Cache

    print_case("chunk-cache")
    c = Chunks(dev, [100, 1, 12], [77, 300, 0], 6, 2, 128, 32, seed=13)
    want = c.run()
    cache = KV8Cache(c.k_cache.shape[0], 2, 128, page_size=32, device=dev)
    cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale = c.k_cache, c.v_cache, c.k_scale, c.v_scale
    assert torch.equal(cache.attend(c.q, c.table, c.seq_lens, c.starts), want)
    with pytest.raises(ValueError, match="workspace"):
        cache.attend(c.q, c.table, c.seq_lens, c.starts, workspace=c.seq_lens)
    out = torch.empty_like(want)
    need = capi.kv8_chunk_attention_scratch_bytes(3, 113, 6, 2, 128, 32, c.table.shape[1])
    scratch = torch.empty(need, dtype=torch.uint8, device=dev)
    assert capi.kv8_chunk_attention(c.q, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens, c.starts, out, scratch,
                                    128 ** -0.5) == capi.LB_OK
    assert torch.equal(out, want)
    # whole and in three pieces over the same pages
    q = torch.randn((177, 6, 128), device=dev).half()
    table, one = c.table[:1].contiguous(), lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    whole = cache.attend(q, table, one([177]), one([0, 177])).float()
    parts, at = [], 0
    for n in (50, 1, 126):
        parts.append(cache.attend(q[at:at + n], table, one([at + n]), one([0, n])).float())
        at += n
    assert (torch.cat(parts) - whole).abs().max() <= 2.0 ** -9 * whole.abs().max()
