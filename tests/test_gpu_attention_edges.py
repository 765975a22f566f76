"""The attention operators where a call is only partly ordinary: absent pages, padding, non-finite and very unequal scales, wide columns.

Oracles and tolerances are those of ``test_gpu_attention.py``; where one is
added here, its derivation stands with it.
"""
from __future__ import annotations

import numpy as np
import pytest

from oracle import attention_oracle as A
from tests.gpu_util import print_case
from tests.test_gpu_attention import AppendCase, Cached, _np

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ append ---

def _rows_near(got, want):
    size = np.abs(want).max() + 1
    return (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -22 * size + 2.0 ** -25).all()


KEYS_OUT = [
    # lens (new tokens included), new, heads_q, heads_kv, d, page, rot, interleaved, pages left out as (sequence, page), table pages
    ([40, 70], [40, 70], 4, 2, 64, 16, 64, False, [(0, 0), (1, 0), (1, 1), (1, 3)], 9),     # only a window keeps its pages
    ([90, 33], [90, 33], 3, 1, 128, 32, 128, True, [(0, 1)], 2),                            # the table ends before the tokens
    ([0, 2, 24, 34, -3], [4, 4, 4, 4, 4], 2, 1, 64, 16, 64, False, [(2, 1), (3, 2)], 4),    # padding: none, some and all of a sequence
    ([7, 19, 130], [20, 40, 130], 2, 2, 256, 64, 64, True, [(2, 0)], 2),
    ([50, 3], [150, 3], 5, 1, 128, 16, 0, False, [(0, 0), (0, 3)], 3),                      # more padding than a page holds
]


@pytest.mark.parametrize("case", range(len(KEYS_OUT)))
@pytest.mark.parametrize("strided,queries", [(False, True), (True, False)])
def test_append_returns_the_keys_of_every_token(dev, case, strided, queries):
    """A token without a page, or past the table, has its rotated key all the same; padding has zeros; a token of no sequence is left out."""
    import langburst_cuda as lc
    import torch

    lens, news, hq, hkv, d, p, rot, inter, absent, width = KEYS_OUT[case]
    print_case("append-keys-out", case, strided, queries)

    made = []
    for _ in range(2):
        torch.manual_seed(case)  # the order of the pages
        made.append(AppendCase(dev, [max(x - n, 0) for x, n in zip(lens, news)], news, hq, hkv, d, p, rot, seed=case, strided=strided,
                               positions=max(lens)))
    c, plain = made
    for x in (c, plain):
        x.seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        for b, page in absent:
            if page < x.table.shape[1]:
                x.table[b, page] = -1 if b else 10 ** 6
        x.table = x.table[:, :width].contiguous()
        if strided and len(set(news)) == 1:
            x.starts = None
    tokens = sum(news)
    k_out = torch.full((tokens, hkv, d), float("nan"), dtype=torch.float16, device=dev)
    q_out = torch.full((tokens, hq, d), float("nan"), dtype=torch.float16, device=dev) if queries else None
    lc.kv8_append_out(c.q if queries else None, c.k, c.v, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens,
                      c.starts, c.rotation, q_out, k_out, inter)
    torch.cuda.synchronize()
    angles, at = None if c.rotation is None else _np(c.rotation), 0
    for b, n in enumerate(news):
        for i in range(n):
            pos = lens[b] - n + i
            for got, x in ((k_out, c.k),) + (((q_out, c.q),) if queries else ()):
                if pos < 0:
                    assert (got[at + i] == 0).all(), (b, i)
                    continue
                want = _np(x[at + i]) if angles is None else A.rotate(_np(x[at + i]), angles[pos, :rot // 2], angles[pos, rot // 2:], inter)
                assert _rows_near(_np(got[at + i]), want), (b, i, pos)
        at += n
    # the cache is what it is without the keys' rows
    lc.kv8_append_out(None, plain.k, plain.v, plain.k_cache, plain.v_cache, plain.k_scale, plain.v_scale, plain.table, plain.seq_lens,
                      plain.starts, plain.rotation, None, None, inter)
    for x, y in ((c.k_cache, plain.k_cache), (c.v_cache, plain.v_cache), (c.k_scale, plain.k_scale), (c.v_scale, plain.v_scale)):
        assert torch.equal(x, y)


def test_append_leaves_the_keys_rows_of_no_sequence(dev):
    import langburst_cuda as lc
    import torch

    print_case("append-keys-out-rest")
    c = AppendCase(dev, [0, 0, 0], [5, 40, 7], 2, 1, 64, 16, 64, seed=1)
    k_out = torch.full((52, 1, 64), 7.0, dtype=torch.float16, device=dev)
    # the last seven tokens are of no sequence
    lc.kv8_append_out(None, c.k, c.v, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table[:2].contiguous(), c.seq_lens[:2].contiguous(),
                      c.starts[:3].contiguous(), c.rotation, None, k_out, False)
    torch.cuda.synchronize()
    assert (k_out[45:] == 7).all() and (k_out[:45] != 7).any(-1).all()


def test_cache_append_returns_keys_that_prompt_attention_can_read(dev):
    """Through the cache object: early pages left out, and the prompt's attention still sees every key."""
    import torch

    from neurova_amd.attention import KV8Cache, prompt_attention, rotation_table

    print_case("append-window-then-prompt")
    hq, hkv, d, n = 4, 2, 128, 100
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    qkv = torch.randn((n, hq + 2 * hkv, d), device=dev, generator=g).half()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    table = rotation_table(n, 64, device=dev)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    whole, window = KV8Cache(8, hkv, d, page_size=16, device=dev), KV8Cache(8, hkv, d, page_size=16, device=dev)
    junk = torch.full((n, hkv, d), float("nan"), dtype=torch.float16, device=dev)
    del junk  # what an allocation may hold
    got = window.append(q, k, v, torch.tensor([[-1, -1, -1, -1, -1, 4, 2]], dtype=torch.int32, device=dev), lens, rotation=table, return_k=True)
    want = whole.append(q, k, v, torch.tensor([[5, 1, 0, 7, 3, 4, 2]], dtype=torch.int32, device=dev), lens, rotation=table, return_k=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(prompt_attention(*got, v), prompt_attention(*want, v))


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_a_sequence_whose_last_tokens_are_not_given(dev, interleaved):
    """cu_seqlens[b + 1] - 1 is a sequence's newest token: one past the given tokens moves none of these, keys or queries."""
    import langburst_cuda as lc
    import torch

    print_case("append-cut-short", interleaved)
    made = []
    for _ in range(2):
        torch.manual_seed(5)
        made.append(AppendCase(dev, [0, 30], [20, 30], 3, 2, 64, 16, 64, seed=6))
    long, short = made
    tokens = 40  # of 50: ten of the second sequence are missing
    outs = []
    for c, lens, starts in ((long, [20, 60], [0, 20, 50]), (short, [20, 50], [0, 20, 40])):
        q, k = (torch.full((tokens, h, 64), float("nan"), dtype=torch.float16, device=dev) for h in (3, 2))
        lc.kv8_append_out(c.q[:tokens], c.k[:tokens], c.v[:tokens], c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table,
                          torch.tensor(lens, dtype=torch.int32, device=dev), torch.tensor(starts, dtype=torch.int32, device=dev),
                          c.rotation, q, k, interleaved)
        outs.append((q, k, c.k_cache, c.v_cache, c.k_scale, c.v_scale))
    torch.cuda.synchronize()
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_append_without_a_single_page(dev):
    """A table of no pages, or a cache of none: nothing is stored, and the rotated rows are there."""
    import langburst_cuda as lc
    import torch

    print_case("append-no-pages")
    for no_pages in (False, True):
        c = AppendCase(dev, [0, 0], [5, 40], 2, 1, 64, 16, 64, seed=1)
        want_q, want_k = (torch.empty((45, h, 64), dtype=torch.float16, device=dev) for h in (2, 1))
        lc.kv8_append_out(c.q, c.k, c.v, c.k_cache, c.v_cache, c.k_scale, c.v_scale, c.table, c.seq_lens, c.starts, c.rotation,
                          want_q, want_k, False)
        q, k = torch.zeros_like(want_q), torch.zeros_like(want_k)
        cache = [torch.empty((0,) + t.shape[1:], dtype=t.dtype, device=dev) for t in (c.k_cache, c.v_cache, c.k_scale, c.v_scale)] if no_pages else [c.k_cache, c.v_cache, c.k_scale, c.v_scale]
        table = c.table if no_pages else torch.empty((2, 0), dtype=torch.int32, device=dev)
        lc.kv8_append_out(c.q, c.k, c.v, *cache, table, c.seq_lens, c.starts, c.rotation, q, k, False)
        torch.cuda.synchronize()
        assert torch.equal(q, want_q) and torch.equal(k, want_k)


# --------------------------------------------------------- attention, cache ---

@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("hq,hkv,d,n", [(4, 2, 64, 3), (12, 2, 64, 4), (6, 2, 128, 3), (10, 1, 128, 4), (6, 1, 256, 3), (24, 2, 256, 3)])
def test_attention_over_the_cache_keeps_non_finite_scales_behind_the_causal_limit(dev, bad, hq, hkv, d, n):
    """A new token's page that is not finite reaches the rows that see a token of it, and no earlier row."""
    import langburst_cuda as lc

    print_case("kv8-attention-masked-scale", bad, hq, hkv, d, n)
    for which in ("v_scale", "k_scale"):
        for length in (16 + n - 1, 304 + n - 1, 2001):  # row 0 is its page's last token; 2001 is one past a page
            c = Cached(dev, [length], n, hq, hkv, d, 16, seed=length)
            last = (length - 1) // 16
            clean = c.run(lc)
            c.check(clean)
            clean = _np(clean)
            getattr(c, which)[int(c.table[0, last])] = bad
            got = _np(c.run(lc))
            for i in range(n):
                if length - n + i < last * 16:  # within the outputs' rounding of the clean call's: fp16 at either side
                    assert (np.abs(got[i] - clean[i]) <= 2.0 ** -10 * np.abs(clean[i]) + 2.0 ** -17 * np.abs(clean[i]).max() + 2.0 ** -24).all(), (which, length, i)
                elif which == "v_scale":
                    assert np.isnan(got[i]).all(), (which, length, i)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 4, 128), (6, 1, 256)])
def test_attention_over_the_cache_shows_an_infinite_key_scale(dev, hq, hkv, d):
    """Keys that are not finite have no scores, below zero or above: every row that sees them is NaN."""
    import langburst_cuda as lc

    print_case("kv8-attention-key-scale", hq, hkv, d)
    for length, page in ((40, 1), (700, 3), (700, 43), (33, 2), (1025, 64)):  # the last two with a single token in the page
        c = Cached(dev, [length], 1, hq, hkv, d, 16, seed=length + page)
        c.k_scale[int(c.table[0, page]), 0] = float("inf")
        got = c.run(lc)
        assert np.isnan(_np(got[:, :hq // hkv])).all()
        if hkv > 1:
            c.check(got, heads=range(1, hkv))


@pytest.mark.parametrize("ratio", [1e-6, 1e-7, 1e-9])
@pytest.mark.parametrize("hq,hkv,d,n", [(4, 4, 64, 1), (10, 1, 64, 2), (4, 1, 128, 1), (12, 1, 128, 2), (6, 1, 256, 1)])
def test_attention_over_the_cache_to_a_page_of_small_values_among_large_ones(dev, ratio, hq, hkv, d, n):
    """Pages that a row ignores do not cost the others' weights their bits, however large their values.

    The page attended to is 28 above the rest in its scores, so all others have
    2^-40 of the weight, and the output is its values' average.  The largest value
    scale is 200: values of the small page stay normal fp16 numbers down to 1e-7.
    """
    import langburst_cuda as lc

    print_case("kv8-attention-small-page", ratio, hq, hkv, d, n)
    length, page = 700, 16
    for target in (0, 19, 43 - n):  # the first page, one in the middle, the last whole one
        c = Cached(dev, [length], n, hq, hkv, d, page, seed=target)
        pages = c.table[0, :-(-length // page)].long()
        small = int(pages[target])
        c.k_scale[pages] = 0.02
        c.v_scale[pages], c.v_scale[small] = 200.0, 200.0 * ratio
        c.k_cache[pages, :, :, 0], c.k_cache[small, :, :, 0] = -127, 127
        c.q.mul_(0.05)[:, :, 0] = 14 / 2.54
        out = c.run(lc, scale=1.0)
        for h in range(hkv):
            k, v, _ = c.keys(0, h)
            for j in range(hq // hkv):
                q = _np(c.q[:, h * (hq // hkv) + j])
                sees = [length - n + i + 1 for i in range(n)]
                want, spread, _ = A.attend(q, k, v, 1.0, sees)
                w = 2 * A.score_error(q, k, 1.0) + 2.0 ** -18
                err = np.abs(_np(out[:, h * (hq // hkv) + j]) - want)
                bad = err > 2.0 ** -11 * np.abs(want) + w * spread + 2.0 ** -25
                assert not bad.any(), (target, h, j, err.max(), np.abs(want).max())


@pytest.mark.parametrize("hq,hkv,d,n", [(4, 2, 64, 3), (12, 1, 128, 3), (6, 1, 256, 5)])
def test_attention_over_the_cache_of_lengths_past_the_table(dev, hq, hkv, d, n):
    """Token i of n sees the keys up to seq_lens - n + i, of which those in the table exist."""
    import langburst_cuda as lc
    import torch

    print_case("kv8-attention-past-table", hq, hkv, d, n)
    for pages in (6, 40):
        for past in (0, 1, n - 1, n, 1000):
            c = Cached(dev, [pages * 16, 50], n, hq, hkv, d, 16, seed=pages + past)
            c.table = c.table[:, :pages].contiguous()
            c.seq_lens = torch.tensor([pages * 16 + past, 50], dtype=torch.int32, device=dev)
            out = c.run(lc)
            for h in range(hkv):
                k, v, _ = c.keys(0, h)
                for j in range(hq // hkv):
                    at = h * (hq // hkv) + j
                    q = _np(c.q[:n, at])
                    want, spread, _ = A.attend(q, k, v, d ** -0.5, [pages * 16 + past - n + i + 1 for i in range(n)])
                    err = np.abs(_np(out[:n, at]) - want)
                    bad = err > 2.0 ** -11 * np.abs(want) + (2 * A.score_error(q, k, d ** -0.5) + 2.0 ** -18) * spread + 2.0 ** -25
                    assert not bad.any(), (pages, past, at, err.max())


def test_attention_over_the_cache_of_lengths_past_the_table_among_many(dev):
    """The lengths are read 64 sequences at a time: one past the table in every part of them."""
    import langburst_cuda as lc
    import torch

    print_case("kv8-attention-past-table-many")
    n, pages, past = 3, 20, 2
    lens = [pages * 16 if b % 37 == 5 else 5 + b % 7 for b in range(150)]
    c = Cached(dev, lens, n, 4, 1, 64, 16, seed=9)
    c.table = c.table[:, :pages].contiguous()
    c.seq_lens = torch.tensor([x + past * (x == pages * 16) for x in lens], dtype=torch.int32, device=dev)
    out = _np(c.run(lc))
    for b, length in enumerate(lens):
        k, v, _ = c.keys(b, 0)
        for h in range(4):
            rows = slice(b * n, (b + 1) * n)
            sees = [length + past * (length == pages * 16) - n + i + 1 for i in range(n)]
            q = _np(c.q[rows, h])
            want, spread, _ = A.attend(q, k, v, 0.125, sees)
            bad = np.abs(out[rows, h] - want) > 2.0 ** -11 * np.abs(want) + (2 * A.score_error(q, k, 0.125) + 2.0 ** -18) * spread + 2.0 ** -25
            assert not bad.any(), (b, h)


WIDE = [
    # lens, n, heads_q, heads_kv, d, page: columns in one block of 16, one of 32, and more blocks, joined by
    # the last worker and by a second launch
    ([5000], 1, 4, 1, 64, 16),                   # 64 channels, 4 columns, second launch
    ([2000, 900, 70], 4, 12, 2, 64, 64),         # 24 columns, ranges of several units
    ([9000, 400], 3, 16, 2, 64, 32),             # 24 columns, second launch
    ([2000, 900], 6, 12, 2, 64, 64),             # 36 columns: two blocks
    ([9000, 33], 6, 16, 2, 64, 128),             # 48 columns: two blocks, second launch
    ([3000, 700, 2000], 5, 8, 2, 128, 16),       # 20 columns
    ([9000], 5, 4, 1, 128, 32),                  # 20 columns, second launch
    ([3000, 700, 5], 9, 8, 2, 128, 16),          # 36 columns: two blocks
    ([9000], 10, 4, 1, 128, 64),                 # 40 columns: two blocks, second launch
    ([6000], 1, 6, 1, 256, 64),                  # second launch
    ([3000, 100], 4, 12, 2, 256, 32),            # 24 columns: two blocks of 16
    ([6000], 4, 12, 1, 256, 64),                 # 48 columns: three blocks, second launch
    ([260, 100], 70, 4, 2, 64, 16),              # 140 columns: five blocks, a sequence with little more than the new tokens
    ([600] * 40, 3, 12, 2, 128, 16),             # 18 columns, about a slot for each worker
    ([1500] * 90, 3, 12, 2, 128, 16),            # and ranges that end inside pairs
    ([300] + [5] * 70 + [2600], 3, 7, 1, 128, 32),  # more sequences than a wave has lanes
]


@pytest.mark.parametrize("case", range(len(WIDE)))
def test_attention_over_the_cache_in_every_form(dev, case):
    import langburst_cuda as lc
    import torch

    print_case("kv8-attention-wide", case, *WIDE[case][1:])
    c = Cached(dev, *WIDE[case], seed=case)
    out = c.run(lc)
    c.check(out, heads=None if len(WIDE[case][0]) < 40 else [0])
    for _ in range(3):
        assert torch.equal(out, c.run(lc)), "repeated calls differ"
