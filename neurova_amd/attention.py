"""The attention between a layer's QKV and O projections: an 8-bit paged cache, its writer and readers.

:class:`KV8Cache` holds one layer's keys and values in 8 bits, in pages of 16
to 128 tokens with one fp32 scale for each page and key/value head.  Which page
holds which tokens of which sequence is the caller's: every call takes a
``page_table`` int32 ``[batch, max_pages]`` and ``seq_lens`` int32 ``[batch]``
(the new tokens included), both on the GPU, so nothing here waits for the
device.  A decode step is

    cache.append(q, k, v, page_table, seq_lens, rotation=table, q_out=q)
    out = cache.attend(q, page_table, seq_lens)

and a batch of prompts, packed one after the other,

    q, k = cache.append(q, k, v, page_table, seq_lens, cu_seqlens, rotation=table, return_k=True)
    out = prompt_attention(q, k, v, cu_seqlens)

Rows are fp16 ``[tokens, heads, head_dim]`` and may be views of the fused QKV
projection's output.  Everything runs on the current stream through the
``langburst_cuda`` ops ``kv8_append_out``, ``kv8_attention_out`` and
``prompt_attention_out``; there is no CPU path.  These are this package's own
operators, without a counterpart in the reference's projection path.
"""
from __future__ import annotations

import math

from .store import _ops, _require_device

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)


def rotation_table(positions: int, rot_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                   original_positions: int | None = None, device="cuda"):
    """cos | sin of every position, fp32 ``[positions, rot_dim]``, as ``KV8Cache.append`` takes it.

    Pair i of a head turns by ``position * base ** (-2 i / rot_dim)``, computed
    in 64 bits.  ``scaling`` stretches a model's positions by ``factor``:

    * ``"linear"``: positions are divided by the factor;
    * ``"ntk"``: the base grows to ``base * factor ** (rot_dim / (rot_dim - 2))``,
      which stretches the slowest pair by the factor and leaves the fastest;
    * ``"yarn"`` (Peng et al., 2023): pairs that turn more than 32 times within
      ``original_positions`` stay, pairs that turn less than once are divided by
      the factor, with a linear ramp between, and cos and sin are multiplied by
      ``0.1 ln(factor) + 1``.
    """
    import torch

    if positions < 0 or rot_dim <= 0 or rot_dim % 16 != 0:
        raise ValueError(f"rot_dim must be a positive multiple of 16 and positions not negative, got {rot_dim} and {positions}")
    if factor <= 0 or base <= 0:
        raise ValueError("base and factor must be positive")
    pair = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "ntk":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = base ** (-pair / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if not original_positions:
            raise ValueError("yarn scaling needs original_positions")

        def pair_that_turns(times: float) -> float:
            return rot_dim * math.log(original_positions / (times * 2 * math.pi)) / (2 * math.log(base))

        low = max(0, math.floor(pair_that_turns(32)))
        high = math.ceil(pair_that_turns(1))
        ramp = ((pair / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * amplitude).float().to(device)


class KV8Cache:
    """One layer's keys and values: int8 codes with an fp32 scale for each page and head.

    ``k_cache`` int8 ``[pages, heads, page_size, head_dim]``, ``v_cache`` int8
    ``[pages, heads, head_dim, page_size]``, ``k_scale`` and ``v_scale`` fp32
    ``[pages, heads]``; a value is its code times its page's scale.  A token
    and head take 2 * head_dim bytes.
    """

    def __init__(self, num_pages: int, heads_kv: int, head_dim: int, page_size: int = 64, device="cuda"):
        import torch

        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        self.page_size = int(page_size)
        self.k_cache = torch.zeros((num_pages, heads_kv, page_size, head_dim), dtype=torch.int8, device=device)
        self.v_cache = torch.zeros((num_pages, heads_kv, head_dim, page_size), dtype=torch.int8, device=device)
        self.k_scale = torch.zeros((num_pages, heads_kv), dtype=torch.float32, device=device)
        self.v_scale = torch.zeros((num_pages, heads_kv), dtype=torch.float32, device=device)
        self._workspaces = {}

    def _buffers(self):
        return self.k_cache, self.v_cache, self.k_scale, self.v_scale

    def append(self, q, k, v, page_table, seq_lens, cu_seqlens=None, *, rotation=None, interleaved: bool = False,
               q_out=None, return_k: bool = False):
        """Rotates ``q`` and ``k`` to their positions and stores ``k`` and ``v``; returns q rotated, or (q, k) rotated.

        ``cu_seqlens`` int32 ``[batch + 1]`` says which of the packed tokens are
        whose; without it every sequence has the same number.  ``rotation`` is a
        :func:`rotation_table` (None: no rotation), ``q_out`` where the rotated
        queries go (it may be ``q`` itself).  With ``return_k`` every token of a
        sequence has its rotated key, with or without a page; padding has zeros.
        A token's page and its scale are described at ``lb_kv8_append`` in
        ``include/langburst_lowbit.h``.
        """
        import torch

        _require_device(k, "KV8Cache.append")
        if q is not None and q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device) if return_k else None
        _ops().kv8_append_out(q, k, v, *self._buffers(), page_table, seq_lens, cu_seqlens, rotation, q_out, k_out, interleaved)
        return (q_out, k_out) if return_k else q_out

    def attend(self, q, page_table, seq_lens, *, scale: float | None = None, out=None, workspace=None):
        """Attention of the newest tokens of every sequence (``q`` holds the same number for each) over its pages.

        The queries of one call see the keys up to their own.  ``scale`` is
        ``head_dim ** -0.5`` by default.  ``workspace`` int32, zeros, of tokens *
        heads entries, is left zero and belongs to calls that run in order; without
        it the cache keeps one for each stream, and a call captured into a graph
        clears one of its own in every replay.
        """
        import torch

        _require_device(q, "KV8Cache.attend")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _ops().kv8_attention_out(q, *self._buffers(), page_table, seq_lens, out, self._workspace(q) if workspace is None else workspace,
                                 q.shape[2] ** -0.5 if scale is None else scale)
        return out

    def _workspace(self, q):
        """A buffer of zeros for each stream, whose calls run in order; in a capture one from the graph's memory, which nothing else may keep."""
        import torch

        need = q.shape[0] * q.shape[1]
        if torch.cuda.is_current_stream_capturing():
            return torch.zeros((need,), dtype=torch.int32, device=q.device)
        key = (q.device.index, torch.cuda.current_stream(q.device).cuda_stream)
        ws = self._workspaces.get(key)
        if ws is None or ws.numel() < need:
            ws = self._workspaces[key] = torch.zeros((max(need, 4096),), dtype=torch.int32, device=q.device)
        return ws


def prompt_attention(q, k, v, cu_seqlens=None, *, scale: float | None = None, out=None):
    """Causal attention inside each packed sequence; ``cu_seqlens`` None: all tokens are one sequence.

    Rows of tokens that belong to no sequence are not written.
    """
    import torch

    _require_device(q, "prompt_attention")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _ops().prompt_attention_out(q, k, v, cu_seqlens, out, q.shape[2] ** -0.5 if scale is None else scale)
    return out
