"""The pages of the 8-bit cache: which sequence holds which, kept on the GPU.

:class:`KV8Pages` is a table of rows (sequences, prompts kept for others) with
the ``page_table`` and ``seq_lens`` that :class:`neurova_amd.attention.KV8Cache`
takes, and the number of rows that hold each page.  A prompt and eight answers:

    pages = KV8Pages(num_pages=4096, rows=64, max_tokens=32768, page_size=64, caches=caches)   # one cache a layer
    pages.extend(prompt, prompt_tokens)                     # int32 row and token numbers, on the GPU
    ... every layer appends the prompt's keys and values ...
    pages.fork(prompt.expand(8).contiguous(), answers)      # nothing is copied
    status = pages.extend(answers, 1)                       # pages for a token each; the prompt's last page is copied
    table = pages.page_table[answers]
    lens = pages.seq_lens[answers] * (status == 0)          # refused: nothing has changed, and the new tokens are padding
    cache.append(q, k, v, table, lens)                      # every layer
    out = cache.attend(q, table, lens)
    pages.free(answers)

A row's lengths do not change when :meth:`KV8Pages.extend` refuses, so tokens
appended by them all the same would overwrite the last ones that the row holds,
and those of every row that shares the page.  Lengths of zero instead store
nothing, and nothing has to wait for the status.

Free pages are handed out lowest first, :meth:`KV8Pages.compact` moves the
pages in use to the front, and nothing waits for the device.  The operators
``kv8_pages_free_out``, ``kv8_pages_fork_out``, ``kv8_pages_extend_out``,
``kv8_pages_compact_out`` and ``kv8_copy_pages`` of ``langburst_cuda`` do the
work on the current stream (``include/langburst_lowbit.h`` says what each
promises); there is no CPU path.  They are this package's own, without a
counterpart in the reference's projection path.
"""
from __future__ import annotations

import operator

from .attention import PAGE_SIZES
from .store import _ops, _require_device


def kv8_layers(caches):
    """What the operators on pages take for the caches (:class:`KV8Cache`) of all layers."""
    caches = list(caches)
    for c in caches:
        _require_device(c.k_cache, "kv8_layers")
    return _ops().KV8Layers(*([getattr(c, name) for c in caches] for name in ("k_cache", "v_cache", "k_scale", "v_scale")))


def copy_pages(layers, src, dst):
    """Copies pages ``src`` to ``dst`` (int32, on the GPU) in every layer; ``layers`` as :func:`kv8_layers` gives them, or the caches.

    A page must not be the destination of two pairs, nor of one and the source of another.
    """
    _ops().kv8_copy_pages(layers if isinstance(layers, _ops().KV8Layers) else kv8_layers(layers), src, dst)


class KV8Pages:
    """Rows of pages: ``page_table`` int32 ``[rows, max_pages]``, ``seq_lens`` int32 ``[rows]``, ``refs`` int32 ``[num_pages]``.

    ``caches``: one :class:`KV8Cache` of ``num_pages`` pages of ``page_size`` tokens
    for each layer.  Without them the tables alone change: nothing is copied or moved,
    and :meth:`extend` refuses rows whose last page would have to be copied.
    ``rows`` arguments are int32 tensors on the GPU, of at most 4096 rows.
    """

    def __init__(self, num_pages: int, rows: int, max_tokens: int, page_size: int = 64, caches=(), device="cuda"):
        import torch

        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if num_pages < 0 or rows < 0 or max_tokens < 0:
            raise ValueError("num_pages, rows and max_tokens must not be negative")
        caches = list(caches)
        for i, c in enumerate(caches):
            if (c.k_cache.shape[0], c.k_cache.shape[2]) != (num_pages, page_size):
                raise ValueError(f"the caches must have {num_pages} pages of {page_size} tokens, "
                                 f"got {c.k_cache.shape[0]} of {c.k_cache.shape[2]} in layer {i}")
        self.page_size = int(page_size)
        self.page_table = torch.full((rows, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros((rows,), dtype=torch.int32, device=device)
        self.refs = torch.zeros((num_pages,), dtype=torch.int32, device=device)
        self.layers = kv8_layers(caches) if caches else None

    def _state(self):
        return self.page_table, self.seq_lens, self.refs, self.page_size

    def _counts(self, n, rows):
        import torch

        if isinstance(n, torch.Tensor):
            return n
        return torch.full(rows.shape, operator.index(n), dtype=torch.int32, device=rows.device)

    def extend(self, rows, new, status=None):
        """Pages for ``new`` more tokens (a number, or int32 for each) of the rows, and their lengths; returns ``status`` int32 ``[1]``.

        0: done.  Otherwise nothing has changed: the number of pages that are
        missing, -1 where a row would pass the end of the table, -2 where a shared
        page would have to be copied and there are no caches.  The tokens must not be
        appended then; ``seq_lens[rows] * (status == 0)`` as the lengths makes padding of them.
        """
        import torch

        _require_device(rows, "KV8Pages.extend")
        if status is None:
            status = torch.empty((1,), dtype=torch.int32, device=rows.device)
        _ops().kv8_pages_extend_out(*self._state(), rows, self._counts(new, rows), status, self.layers)
        return status

    def fork(self, parents, children, lens=None, done=None):
        """Each empty row of ``children`` becomes its parent's first ``lens`` tokens (all of them by default), by sharing pages.

        A child that holds tokens, or that is named again, is left as it is; ``done`` int32 says 1 for the others.
        """
        _require_device(parents, "KV8Pages.fork")
        _ops().kv8_pages_fork_out(*self._state(), parents, children, None if lens is None else self._counts(lens, parents), done)

    def free(self, rows, keep=None):
        """The rows keep their first ``keep`` tokens (none by default) and give up the pages behind them."""
        _require_device(rows, "KV8Pages.free")
        _ops().kv8_pages_free_out(*self._state(), rows, None if keep is None else self._counts(keep, rows))

    def compact(self, used=None):
        """Moves the pages in use to the front of the pool, in every layer; returns their number, int32 ``[1]``."""
        import torch

        _require_device(self.refs, "KV8Pages.compact")
        if used is None:
            used = torch.empty((1,), dtype=torch.int32, device=self.refs.device)
        _ops().kv8_pages_compact_out(self.page_table, self.refs, used, self.layers)
        return used
