"""What the GPU tests of serving would notice, shown on the CPU: mistakes planted in the expected values, and which calls their draws make."""
from __future__ import annotations

import pytest

from tests.test_gpu_kv8_pages import Model
from tests.test_gpu_kv8_serving_edges import SCALED, Calls, Scaled


@pytest.mark.parametrize("d,p,spread,kinds", SCALED)
def test_a_wrong_scale_is_noticed(d, p, spread, kinds):
    import torch

    s = Scaled(d, p, spread, seed=d + int(spread), kinds=kinds)
    s.has_power()
    right = torch.zeros(s.c.q.shape, dtype=torch.float64)
    for _, h, rows, want, _ in s.wanted():
        right[rows, h] = want
    s.check(right.half())
    with pytest.raises(AssertionError):
        s.check(torch.zeros_like(right).half())
    # of each sequence's first page: values 5 % off, the keys' sign
    first = torch.from_numpy(s.c.table_np[:, 0]).long()
    for change in (lambda c: c.v_scale.index_copy_(0, first, c.v_scale[first] * 1.05), lambda c: c.k_scale.index_copy_(0, first, -c.k_scale[first])):
        wrong = Scaled(d, p, spread, seed=d + int(spread), kinds=kinds)
        change(wrong.c)
        got = right.clone()
        for _, h, rows, want, _ in wrong.wanted():
            got[rows, h] = want
        with pytest.raises(AssertionError):
            s.check(got.half())


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("seed", range(3))
def test_the_calls_drawn_make_everything_happen(page, seed):
    calls = Calls(seed, page)
    model = Model(calls.pages, calls.rows, calls.width, page)
    for _ in range(80):
        what, args = calls.next(model)
        before = list(model.was)
        calls.count(what, args, getattr(model, what)(*args), before, model)
    calls.enough()
