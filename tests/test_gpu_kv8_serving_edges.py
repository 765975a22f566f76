"""Serving from the 8-bit pages where it can go wrong: refused steps, scales far apart, any order of calls."""
from __future__ import annotations

import re
import textwrap

import pytest

from tests.gpu_util import print_case

pytestmark = pytest.mark.gpu


def documented_step():
    """The decode step of the example in the documentation of ``neurova_amd.pages``: what stands between the fork and the end."""
    from neurova_amd import pages

    block = re.search(r"^ {4}pages\.fork\(.*?\n(.*?)^ {4}pages\.free\(", pages.__doc__, re.S | re.M).group(1)
    return compile(textwrap.dedent(block), "step", "exec")


@pytest.mark.parametrize("refused", ["a page for a copy", "a new page", "the end of a row"])
def test_a_refused_step_as_documented_changes_nothing(dev, refused):
    import torch

    from neurova_amd.attention import KV8Cache
    from neurova_amd.pages import KV8Pages

    print_case("serving-refused", refused)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    held = {"a page for a copy": 21, "a new page": 32, "the end of a row": 48}[refused]
    count, hq, hkv, d = 3, 4, 2, 64
    cache = KV8Cache(4, hkv, d, page_size=16, device=dev)
    pages = KV8Pages(4, 5, 48, page_size=16, caches=[cache], device=dev)
    g = torch.Generator(device=dev)
    g.manual_seed(held)
    rows = lambda n, h: torch.randn((n, h, d), device=dev, generator=g).half()  # noqa: E731
    assert int(pages.extend(i32([0]), held)) == 0
    cache.append(None, rows(held, hkv), rows(held, hkv), pages.page_table[:1], pages.seq_lens[:1], i32([0, held]))
    answers = i32([1, 2, 3])
    pages.fork(i32([0] * count), answers)
    if refused != "the end of a row":
        assert int(pages.extend(i32([4]), 16 if held == 32 else 32)) == 0   # the pool is all but full
    state = [pages.page_table, pages.seq_lens, pages.refs, *cache._buffers()]
    before = [t.clone() for t in state]
    got = {"pages": pages, "cache": cache, "answers": answers, "q": rows(count, hq), "k": 9 * rows(count, hkv), "v": 9 * rows(count, hkv)}
    exec(documented_step(), got)
    assert int(got["status"]) == {"a page for a copy": 3, "a new page": 2, "the end of a row": -1}[refused]
    for now, then in zip(state, before):
        assert torch.equal(now, then)
    assert (got["out"] == 0).all()
    # by the lengths that the table has, the same tokens land on the ones that the rows share
    cache.append(None, got["k"][:1], got["v"][:1], got["table"][:1], pages.seq_lens[answers[:1]])
    assert not torch.equal(cache.k_cache, before[3])
    # and with a row ended, the step goes through
    pages.free(i32([0, 4, 3]))
    got["answers"], got["q"], got["k"], got["v"] = answers[:1], got["q"][:1], got["k"][:1], got["v"][:1]
    pages.free(answers[1:2], i32([16]))
    if refused == "the end of a row":
        pages.free(answers[:1], i32([40]))
    exec(documented_step(), got)
    assert int(got["status"]) == 0 and got["out"].any()
