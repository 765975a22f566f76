"""A small server's steps over the 8-bit pages: prompts arrive in pieces, answers branch from them, rows end and the pool is compacted.

The layers are those of ``attention_layer.py``; one ``KV8Pages`` says for all of
them which row holds which pages.  Every step takes any number of new tokens of
any rows, packed one after the other.

    python examples/serving.py [--layers 2] [--prompts 700 90 1500] [--piece 512] [--answers 4] [--steps 8]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

if __package__ in (None, ""):  # run from a checkout
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from examples.attention_layer import AttentionLayer  # noqa: E402
from neurova_amd.pages import KV8Pages  # noqa: E402


class Server:
    def __init__(self, layers=2, pages=512, rows=32, max_tokens=4096, page_size=16, seed=0, device="cuda", **shape):
        self.layers = [AttentionLayer(pages=pages, page_size=page_size, positions=max_tokens, seed=seed + i, device=device, **shape)
                       for i in range(layers)]
        self.pages = KV8Pages(pages, rows, max_tokens, page_size=page_size, caches=[x.cache for x in self.layers], device=device)
        self.device = device

    def rows(self, numbers):
        return torch.tensor(numbers, dtype=torch.int32, device=self.device)

    def step(self, x, rows, new):
        """x [tokens, hidden]: the ``new`` (numbers) next tokens of the ``rows`` (int32), one row after the other; their hidden states."""
        count = self.rows(new)
        status = self.pages.extend(rows, count)
        starts = torch.zeros(len(new) + 1, dtype=torch.int32, device=self.device)
        torch.cumsum(count, 0, out=starts[1:])
        # a call that found no pages changed nothing: its tokens are padding then, and their states zeros
        table = self.pages.page_table.index_select(0, rows)
        lens = self.pages.seq_lens.index_select(0, rows) * (status == 0)
        for layer in self.layers:
            q, k, v = layer.project(x)
            q = layer.cache.append(q, k, v, table, lens, starts, rotation=layer.rotation, q_out=q)
            x = x + layer.output(layer.cache.attend(q, table, lens, starts))
        return x, status


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prompts", type=int, nargs="+", default=[700, 90, 1500])
    ap.add_argument("--piece", type=int, default=512)
    ap.add_argument("--answers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args(argv)
    n = len(a.prompts)
    longest = max(a.prompts) + a.steps + 1
    per = -(-longest // 16) + 1
    server = Server(a.layers, pages=n * (a.answers + 1) * per, rows=n * (a.answers + 1), max_tokens=longest)
    hidden = server.layers[0].hidden
    state = lambda tokens: torch.randn((tokens, hidden), device="cuda").half()  # noqa: E731

    left, finite = list(a.prompts), True
    while any(left):  # a piece of every prompt that has one left
        new = [min(x, a.piece) for x in left]
        y, status = server.step(state(sum(new)), server.rows(range(n)), new)
        left = [x - t for x, t in zip(left, new)]
        finite = finite and bool(y.isfinite().all()) and int(status) == 0
    # answers share their prompt's pages until they add tokens
    children = server.rows(range(n, n * (a.answers + 1)))
    server.pages.fork(server.rows(range(n)).repeat_interleave(a.answers), children)
    shared = int((server.pages.refs > 0).sum())
    for _ in range(a.steps):
        y, status = server.step(state(children.numel()), children, [1] * children.numel())
        finite = finite and bool(y.isfinite().all()) and int(status) == 0
    held = int((server.pages.refs > 0).sum())
    server.pages.free(children[::2].contiguous())
    server.pages.free(server.rows(range(n)))
    used = int(server.pages.compact())
    y, status = server.step(state(children[1::2].numel()), children[1::2].contiguous(), [1] * children[1::2].numel())
    finite = finite and bool(y.isfinite().all()) and int(status) == 0
    top = int(server.pages.page_table.max())
    print(f"{n} prompts of {sum(a.prompts)} tokens in {shared} pages; {children.numel()} answers of {a.steps} tokens: {held}; "
          f"after half of them ended and the pool was compacted {used}, the highest {top}; finite: {finite}")
    return 0 if finite else 1


if __name__ == "__main__":
    sys.exit(main())
