"""The plan of the attention over the cache, without a GPU (``lb_kv8_attention_describe_plan``)."""
from __future__ import annotations

import pytest

from neurova_amd import capi
from tests.test_gpu_attention import CACHED
from tests.test_gpu_attention_edges import WIDE


@pytest.fixture(scope="module")
def plan(built):
    return capi.kv8_attention_describe_plan


def _form(plan, lens, n, hq, hkv, d, p):
    """Which kernels a case of the GPU tests runs: its table is two pages wider than its longest sequence."""
    width = max([1] + [-(-x // p) for x in lens]) + 2
    r = plan(len(lens), len(lens) * n, hq, hkv, d, p, width)
    return d, r["columns"], r["column_blocks"] > 1, r["launches"]


def test_the_gpu_cases_reach_every_form(plan):
    """Channels, columns of a workgroup, one column block or several, and either join: each that a plan can choose is run."""
    possible = set()
    for d in (64, 128, 256):
        for cols in (1, 16, 17, 32, 33, 100):
            for width in (1, 2, 16, 64, 600):
                for batch in (1, 40):
                    r = plan(batch, batch, cols, 1, d, 128, width)
                    possible.add((d, r["columns"], r["column_blocks"] > 1, r["launches"]))
    assert len(possible) == 16  # 64 and 128 channels: 16 columns, 32, several blocks of 32; 256: 16 and several blocks; twice
    reached = {_form(plan, *c) for c in CACHED + WIDE}
    assert reached == possible


def test_plan_sizes(plan):
    r = plan(1, 1, 40, 8, 128, 64, 64)
    assert r["columns"] == 16 and r["column_blocks"] == 1 and r["workspace_entries"] == 8
    assert r["scratch_bytes"] == capi.kv8_attention_scratch_bytes(1, 1, 40, 8, 128, 64, 64)
    assert plan(1, 4, 40, 8, 128, 64, 64)["columns"] == 32          # 20 columns
    assert plan(1, 4, 24, 4, 256, 64, 64)["column_blocks"] == 2     # 24 columns of 16
    assert plan(0, 0, 4, 2, 64, 16, 4) == dict.fromkeys(capi.KV8_PLAN_FIELDS, 0)
    for bad in ((2, 3, 4, 2, 128, 16, 4), (1, 1, 3, 2, 128, 16, 4), (1, 1, 4, 2, 96, 16, 4), (1, 1, 4, 2, 64, 48, 4)):
        with pytest.raises(ValueError):
            plan(*bad)
