"""What KV8Pages refuses, and takes, before a GPU is asked."""
from __future__ import annotations

import numpy as np
import pytest

from neurova_amd.attention import KV8Cache
from neurova_amd.pages import KV8Pages


def test_caches_of_another_pool_are_refused(built):
    right, fewer, longer = (KV8Cache(n, 2, 64, page_size=p, device="cpu") for n, p in ((8, 16), (7, 16), (8, 32)))
    for caches in ([fewer], [right, fewer], (c for c in [right, longer])):
        with pytest.raises(ValueError, match="8 pages of 16 tokens"):
            KV8Pages(8, 2, 100, page_size=16, caches=caches, device="cpu")
    with pytest.raises(RuntimeError, match="on the GPU"):   # the right ones are passed on
        KV8Pages(8, 2, 100, page_size=16, caches=(c for c in [right]), device="cpu")


def test_counts_are_any_whole_number():
    import torch

    pages, rows = KV8Pages(8, 2, 100, page_size=16, device="cpu"), torch.tensor([0, 1], dtype=torch.int32)
    for n in (3, np.int64(3), np.uint8(3), torch.tensor([3, 3], dtype=torch.int32)):
        got = pages._counts(n, rows)
        assert got.dtype == torch.int32 and got.tolist() == [3, 3]
    for n in (3.0, np.float32(3), "3"):
        with pytest.raises(TypeError):
            pages._counts(n, rows)
