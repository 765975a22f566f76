"""Serving from the 8-bit pages without a GPU: argument checks of the C entry points and scratch sizes."""
from __future__ import annotations

import math

import pytest

from neurova_amd import capi

FAKE = 0x10000  # aligned, never dereferenced: validation fails or returns first
MIS = 0x10002


def _gpu_present() -> bool:
    import torch

    return torch.cuda.is_available()


host_only = pytest.mark.skipif(_gpu_present(), reason="host-side validation checks use fake device pointers")


@pytest.fixture(scope="module")
def L(built):
    return capi.lib()


def _chunk(L, q=FAKE, kc=FAKE, pages=8, p=16, width=400, stride=400, lens=FAKE, cu=FAKE, batch=2, tokens=7, hq=4, hkv=2, d=128,
           out=FAKE, o_stride=512, scale=0.1, scratch=FAKE, nbytes=1 << 40):
    return L.lb_kv8_chunk_attention(q, 512, 128, kc, FAKE, FAKE, FAKE, pages, p, FAKE, width, stride, lens, cu, batch, tokens, hq, hkv,
                                    d, out, o_stride, 128, scale, scratch, nbytes, None)


@host_only
def test_chunk_rejections(L):
    arg, shape, align, scratch = capi.LB_ERR_ARG, capi.LB_ERR_PROB_SHAPE, capi.LB_ERR_ALIGN, capi.LB_ERR_SCRATCH
    assert _chunk(L, batch=0) == capi.LB_OK and _chunk(L, tokens=0) == capi.LB_OK
    assert _chunk(L, hq=3) == arg and _chunk(L, hkv=0) == arg and _chunk(L, stride=399) == arg and _chunk(L, tokens=-1) == arg
    assert _chunk(L, d=96) == shape and _chunk(L, p=24) == shape and _chunk(L, p=256) == shape
    for s in (0.0, -1.0, math.inf, math.nan):
        assert _chunk(L, scale=s) == arg
    assert _chunk(L, q=None) == arg and _chunk(L, out=None) == arg and _chunk(L, kc=None) == arg
    assert _chunk(L, lens=None) == arg and _chunk(L, cu=None) == arg
    assert _chunk(L, q=MIS) == align and _chunk(L, kc=MIS) == align and _chunk(L, scratch=MIS) == align
    assert _chunk(L, o_stride=516) == align
    assert _chunk(L, scratch=None, nbytes=0) == scratch and _chunk(L, nbytes=64) == scratch
    assert _chunk(L, pages=1 << 31) == arg and _chunk(L, tokens=1 << 25) == arg
    # work is numbered in 32 bits
    assert _chunk(L, batch=1 << 20, tokens=1 << 24, width=1 << 20, stride=1 << 20) == shape


def test_chunk_scratch_sizes(L):
    f = L.lb_kv8_chunk_attention_scratch_bytes
    assert f(0, 0, 4, 2, 128, 16, 400) == 0 and f(2, 7, 4, 2, 100, 16, 400) == 0 and f(2, 7, 5, 2, 128, 16, 400) == 0
    assert f(2, 7, 4, 2, 128, 16, 1) == 0  # one tile of keys: nothing is cut
    short, long = f(1, 64, 40, 8, 128, 16, 64), f(64, 4096, 40, 8, 128, 16, 8192)
    assert 0 < short < long and short % 256 == 0
    assert long <= 256 * 2 * 2 * 128 * 130 * 4 + 256  # two parts for each workgroup that runs at once


def test_host_tensors_are_refused(built):
    import torch

    import neurova_amd
    from neurova_amd.attention import KV8Cache

    lc = neurova_amd.load_extension()
    x = torch.zeros((4, 2, 64), dtype=torch.float16)
    cache = KV8Cache(2, 2, 64, page_size=16, device="cpu")
    table, lens, cu = torch.zeros((1, 2), dtype=torch.int32), torch.tensor([4], dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        cache.attend(x, table, lens, cu)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        lc.kv8_chunk_attention_out(x, cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale, table, lens, cu, x, 0.125)
