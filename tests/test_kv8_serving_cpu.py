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
    assert long <= 256 * 2 * 4 * 128 * 130 * 4 + 512  # four parts for each workgroup that runs at once, and the plan


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


def _extend(L, table=FAKE, rows=4, width=8, stride=8, lens=FAKE, refs=FAKE, pages=32, p=16, which=FAKE, add=FAKE, count=2, status=FAKE,
            layers=None, n_layers=0, heads=2, d=64, scratch=FAKE, nbytes=1 << 20):
    return L.lb_kv8_pages_extend(table, rows, width, stride, lens, refs, pages, p, which, add, count, status, layers, n_layers, heads, d,
                                 scratch, nbytes, None)


@host_only
def test_pages_rejections(L):
    ok, arg, shape, align, scratch = capi.LB_OK, capi.LB_ERR_ARG, capi.LB_ERR_PROB_SHAPE, capi.LB_ERR_ALIGN, capi.LB_ERR_SCRATCH
    free = lambda table=FAKE, lens=FAKE, refs=FAKE, p=16, which=FAKE, count=2, stride=8, rows=4, pages=32: L.lb_kv8_pages_free(  # noqa: E731
        table, rows, 8, stride, lens, refs, pages, p, which, None, count, None)
    assert free(count=0) == ok and free(rows=0, table=None, lens=None) == ok
    assert free(count=-1) == arg and free(count=4097) == arg and free(which=None) == arg
    assert free(table=None) == arg and free(lens=None) == arg and free(refs=None) == arg and free(stride=7) == arg
    assert free(p=20) == shape and free(refs=MIS) == align and free(rows=1 << 31) == arg and free(pages=1 << 31) == arg
    fork = lambda a=FAKE, b=FAKE, count=2: L.lb_kv8_pages_fork(FAKE, 4, 8, 8, FAKE, FAKE, 32, 16, a, b, None, None, count, None)  # noqa: E731
    assert fork(count=0) == ok and fork(a=None) == arg and fork(b=None) == arg and fork(count=4097) == arg
    assert _extend(L, count=-1) == arg and _extend(L, add=None) == arg and _extend(L, status=None) == arg
    assert _extend(L, scratch=MIS) == align and _extend(L, scratch=None) == scratch and _extend(L, nbytes=64) == scratch
    assert _extend(L, n_layers=1) == arg and _extend(L, n_layers=-1) == arg
    assert _extend(L, count=4096, rows=4096, width=1 << 20, stride=1 << 20) == shape   # new pages are numbered in 32 bits
    layer = (capi.KV8Layer * 1)(capi.KV8Layer(FAKE, FAKE, FAKE, FAKE))
    assert _extend(L, layers=layer, n_layers=1, d=96) == shape and _extend(L, layers=layer, n_layers=1, heads=0) == arg
    half = (capi.KV8Layer * 1)(capi.KV8Layer(FAKE, MIS, FAKE, FAKE))
    assert _extend(L, layers=half, n_layers=1) == align
    none = (capi.KV8Layer * 1)(capi.KV8Layer(FAKE, FAKE, None, FAKE))
    assert _extend(L, layers=none, n_layers=1) == arg
    compact = lambda used=FAKE, nbytes=1 << 20: L.lb_kv8_pages_compact(FAKE, 4, 8, 8, FAKE, 32, used, None, 0, 0, 16, 0, FAKE, nbytes, None)  # noqa: E731
    assert compact(used=None) == arg and compact(nbytes=16) == scratch
    copy = lambda layers=layer, n=1, src=FAKE, count=0: L.lb_kv8_copy_pages(layers, n, 32, 2, 16, 64, src, FAKE, count, None)  # noqa: E731
    assert copy() == ok and copy(count=1, src=None) == arg and copy(layers=None) == arg and copy(count=-1) == arg
    assert copy(layers=None, n=0, count=3) == ok


def test_pages_scratch_sizes(L):
    assert L.lb_kv8_pages_extend_scratch_bytes(-1) == 0 and L.lb_kv8_pages_compact_scratch_bytes(-1) == 0
    assert L.lb_kv8_pages_extend_scratch_bytes(1000) % 256 == 0 and L.lb_kv8_pages_extend_scratch_bytes(1000) >= 4000 + 8 * 4096
    assert L.lb_kv8_pages_compact_scratch_bytes(1000) % 256 == 0 and L.lb_kv8_pages_compact_scratch_bytes(1000) >= 12000


def test_pages_on_the_host_are_refused(built):
    import torch

    import neurova_amd
    from neurova_amd.attention import KV8Cache
    from neurova_amd.pages import KV8Pages, kv8_layers

    lc = neurova_amd.load_extension()
    cache, one = KV8Cache(8, 2, 64, page_size=16, device="cpu"), torch.tensor([0], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        kv8_layers([cache])
    with pytest.raises(RuntimeError, match="must be CUDA"):
        lc.KV8Layers([cache.k_cache], [cache.v_cache], [cache.k_scale], [cache.v_scale])
    with pytest.raises(RuntimeError, match="at least one layer"):
        lc.KV8Layers([], [], [], [])
    pages = KV8Pages(8, 2, 100, page_size=16, device="cpu")
    assert pages.page_table.shape == (2, 7) and (pages.page_table == -1).all()
    for call in (lambda: pages.extend(one, 3), lambda: pages.fork(one, one), lambda: pages.free(one), pages.compact):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call()
    with pytest.raises(RuntimeError, match="must be CUDA"):
        lc.kv8_pages_free_out(*pages._state(), one, None)
    with pytest.raises(ValueError, match="negative"):
        KV8Pages(-1, 2, 100, page_size=16, device="cpu")
