"""The scratch of the attention of chunks holds the parts that a plan can have, and not many more."""
from __future__ import annotations

import pytest

from neurova_amd import capi


def _parts(batch, tokens, hq, hkv, d, page, width):
    part = 128 * (d + 2) * 4
    return capi.kv8_chunk_attention_scratch_bytes(batch, tokens, hq, hkv, d, page, width) // part


@pytest.mark.parametrize("d,workers", [(64, 512), (128, 512), (256, 256)])
def test_parts_of_few_and_many_row_blocks(built, d, workers):
    # a few tokens and a wide table: a part for each worker and row block, where these are more than 25 for each row block
    for group in (1, 5, 8):
        blocks = (24 * group // 128 + 1) * 4
        assert workers <= _parts(1, 24, 4 * group, 4, d, 64, 512) <= max(25 * blocks, workers + blocks + 1) + 1
    # many row blocks: what they can be cut into
    assert _parts(8, 8000, 40, 8, d, 64, 512) == 4 * workers
    # a short table: no more than its tiles by two
    assert _parts(1, 24, 4, 4, d, 64, 6) == 4 * 3
