"""The attention operators without a GPU: argument checks of the C entry points, scratch sizes and rotation tables."""
from __future__ import annotations

import math

import numpy as np
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


def _append(L, q=FAKE, k=FAKE, v=FAKE, qo=FAKE, ko=None, kc=FAKE, pages=8, p=16, width=4, stride=4, lens=FAKE, cu=None,
            batch=2, tokens=0, hq=4, hkv=2, d=128, table=FAKE, positions=100, rot=64, ks=FAKE, q_stride=512):
    return L.lb_kv8_append(q, q_stride, 128, k, 256, 128, v, 256, 128, qo, 512, 128, ko, 256, 128, kc, FAKE, ks, FAKE, pages, p,
                           FAKE, width, stride, lens, cu, batch, tokens, hq, hkv, d, table, positions, rot, 0, None)


@host_only
def test_append_rejections(L):
    ok, arg, shape, align = capi.LB_OK, capi.LB_ERR_ARG, capi.LB_ERR_PROB_SHAPE, capi.LB_ERR_ALIGN
    assert _append(L) == ok and _append(L, batch=0, tokens=0) == ok   # nothing to append
    assert _append(L, tokens=3) == arg                                 # 3 tokens of 2 sequences without cu_seqlens
    assert _append(L, tokens=-1) == arg and _append(L, hkv=0) == arg and _append(L, stride=3) == arg
    assert _append(L, d=96) == shape and _append(L, p=24) == shape and _append(L, p=256) == shape
    assert _append(L, rot=24) == shape and _append(L, rot=144) == shape
    assert _append(L, tokens=2, k=None) == arg and _append(L, tokens=2, q=None) == arg
    assert _append(L, tokens=2, table=None) == arg and _append(L, tokens=2, ks=None) == arg
    assert _append(L, tokens=2, lens=None) == arg
    assert _append(L, tokens=2, ko=FAKE) == arg                        # k_out is k
    assert _append(L, tokens=2, k=MIS) == align and _append(L, tokens=2, q_stride=513) == align


def _attend(L, q=FAKE, kc=FAKE, pages=8, p=16, width=4, stride=4, lens=FAKE, batch=2, tokens=2, hq=4, hkv=2, d=128, out=FAKE,
            scale=0.1, ws=FAKE, ws_len=64, scratch=FAKE, nbytes=1 << 30):
    return L.lb_kv8_attention(q, 512, 128, kc, FAKE, FAKE, FAKE, pages, p, FAKE, width, stride, lens, batch, tokens, hq, hkv, d,
                              out, 512, 128, scale, ws, ws_len, scratch, nbytes, None)


@host_only
def test_attention_rejections(L):
    arg, shape, align = capi.LB_ERR_ARG, capi.LB_ERR_PROB_SHAPE, capi.LB_ERR_ALIGN
    assert _attend(L, batch=0, tokens=0) == capi.LB_OK and _attend(L, tokens=0) == capi.LB_OK
    assert _attend(L, tokens=3) == arg and _attend(L, hq=3) == arg and _attend(L, stride=3) == arg
    assert _attend(L, d=80) == shape and _attend(L, p=48) == shape
    assert _attend(L, scale=0.0) == arg and _attend(L, scale=-1.0) == arg and _attend(L, scale=math.inf) == arg
    assert _attend(L, scale=math.nan) == arg
    assert _attend(L, q=None) == arg and _attend(L, kc=None) == arg and _attend(L, lens=None) == arg and _attend(L, ws=None) == arg
    assert _attend(L, q=MIS) == align and _attend(L, scratch=MIS) == align
    assert _attend(L, ws_len=3) == capi.LB_ERR_WORKSPACE
    assert _attend(L, nbytes=16) == capi.LB_ERR_SCRATCH and _attend(L, scratch=None, nbytes=0) == capi.LB_ERR_SCRATCH
    assert _attend(L, batch=1 << 20, tokens=1 << 20, hkv=64, hq=64, width=1 << 20, stride=1 << 20) == shape  # work numbered in 32 bits


@host_only
def test_prompt_rejections(L):
    def prompt(q=FAKE, k=FAKE, cu=None, batch=1, tokens=4, hq=4, hkv=2, d=128, scale=0.1, stride=256):
        return L.lb_prompt_attention(q, 512, 128, k, stride, 128, FAKE, 256, 128, cu, batch, tokens, hq, hkv, d, FAKE, 512, 128,
                                     scale, None)

    arg, shape, align = capi.LB_ERR_ARG, capi.LB_ERR_PROB_SHAPE, capi.LB_ERR_ALIGN
    assert prompt(tokens=0) == capi.LB_OK and prompt(batch=0, tokens=0) == capi.LB_OK
    assert prompt(batch=2) == arg                    # several sequences need cu_seqlens
    assert prompt(hq=5) == arg and prompt(tokens=-1) == arg and prompt(scale=0.0) == arg and prompt(scale=math.nan) == arg
    assert prompt(d=32) == shape and prompt(q=None) == arg and prompt(k=MIS) == align and prompt(stride=260) == align
    assert prompt(stride=1 << 24) == arg             # a tile's offsets are 32-bit


def test_attention_scratch_sizes(L):
    f = L.lb_kv8_attention_scratch_bytes
    assert f(0, 0, 4, 2, 128, 16, 4) == 0 and f(2, 3, 4, 2, 128, 16, 4) == 0 and f(2, 2, 4, 2, 100, 16, 4) == 0
    one, long, wide = f(1, 1, 4, 2, 128, 64, 1), f(1, 1, 4, 2, 128, 64, 4096), f(1, 16, 4, 2, 128, 64, 4096)
    assert 0 < one < min(long, wide) and long % 256 == 0 and wide % 256 == 0


def test_host_tensors_are_refused(built):
    import torch

    import neurova_amd
    from neurova_amd.attention import KV8Cache, prompt_attention

    lc = neurova_amd.load_extension()
    x = torch.zeros((4, 2, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        lc.prompt_attention_out(x, x, x, None, x, 0.125)
    with pytest.raises(RuntimeError, match="on the GPU"):
        prompt_attention(x, x, x)
    cache = KV8Cache(2, 2, 64, page_size=16, device="cpu")
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        cache.append(x, x, x, table, lens)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        lc.kv8_append_out(x, x, x, cache.k_cache, cache.v_cache, cache.k_scale, cache.v_scale, table, lens, None, None, x.clone(),
                          None)
    with pytest.raises(ValueError, match="page_size"):
        KV8Cache(2, 2, 64, page_size=48, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        KV8Cache(2, 2, 96, device="cpu")


def test_rotation_tables():
    from neurova_amd.attention import rotation_table

    t = rotation_table(50, 64, device="cpu").double().numpy()
    angle = np.arange(50)[:, None] * 10000.0 ** (-np.arange(32) / 32)
    assert np.abs(t[:, :32] - np.cos(angle)).max() < 2.0 ** -24 and np.abs(t[:, 32:] - np.sin(angle)).max() < 2.0 ** -24
    # interpolated positions: position 4 p turns as p did
    lin = rotation_table(200, 64, scaling="linear", factor=4, device="cpu").double().numpy()
    assert np.abs(lin[::4] - t).max() < 2.0 ** -22
    # the base that stretches the slowest pair by the factor and leaves the fastest
    ntk = rotation_table(3, 64, scaling="ntk", factor=8, device="cpu").double().numpy()
    assert abs(ntk[1, 0] - np.cos(1.0)) < 1e-6 and abs(ntk[1, 63] - np.sin(10000.0 ** (-31 / 32) / 8)) < 1e-9
    # fast pairs as they were, slow pairs interpolated, both times the amplitude
    yarn = rotation_table(3, 64, scaling="yarn", factor=4, original_positions=4096, device="cpu").double().numpy()
    amp = 0.1 * math.log(4) + 1
    assert abs(yarn[1, 0] - amp * np.cos(1.0)) < 1e-6 and abs(yarn[1, 63] - amp * np.sin(10000.0 ** (-31 / 32) / 4)) < 1e-9
    # long positions keep their precision: the angle is formed in 64 bits
    far = rotation_table(1 << 20, 16, device="cpu")[-1].double().numpy()
    a = ((1 << 20) - 1) * 10000.0 ** (-np.arange(8) / 8)
    assert np.abs(far[:8] - np.cos(a)).max() < 2.0 ** -23
    for bad in (dict(rot_dim=24), dict(rot_dim=0), dict(rot_dim=64, scaling="other"), dict(rot_dim=64, scaling="yarn", factor=2),
                dict(rot_dim=64, factor=0)):
        with pytest.raises(ValueError):
            rotation_table(10, bad.pop("rot_dim"), device="cpu", **bad)
