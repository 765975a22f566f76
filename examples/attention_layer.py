"""One attention layer from hidden states to hidden states: QKV projection, rotation and cache append, attention, O projection.

A batch of packed prompts goes through the layer first (prompt attention beside
the cache's writer), then tokens one by one (attention over the 8-bit cache).
Both projections are Marlin W4A16 tensors of random codes.

    python examples/attention_layer.py [--prompts 300 41 1000] [--steps 8]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

if __package__ in (None, ""):  # run from a checkout
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from neurova_amd.attention import KV8Cache, prompt_attention, rotation_table  # noqa: E402
from neurova_amd.ops import cuda_ops  # noqa: E402


def random_marlin(k: int, n: int, generator, device):
    """qweight int32 [k/16, 2n] of uniform codes and scales fp16 [k/128, n] that keep a product's outputs near unit size."""
    q = torch.randint(-2 ** 31, 2 ** 31, (k // 16, 2 * n), dtype=torch.int32, device=device, generator=generator)
    s = torch.rand((k // 128, n), device=device, generator=generator).add_(0.5).mul_(0.2 / k ** 0.5).half()
    return q, s


class AttentionLayer:
    def __init__(self, hidden=5120, heads=40, heads_kv=8, head_dim=128, pages=256, page_size=16, positions=4096, seed=0, device="cuda"):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.hidden, self.heads, self.heads_kv, self.head_dim = hidden, heads, heads_kv, head_dim
        self.qkv = random_marlin(hidden, (heads + 2 * heads_kv) * head_dim, g, device)
        self.o = random_marlin(heads * head_dim, hidden, g, device)
        self.rotation = rotation_table(positions, head_dim, device=device)
        self.cache = KV8Cache(pages, heads_kv, head_dim, page_size=page_size, device=device)
        self.ops = cuda_ops()

    def project(self, x):
        """q, k, v of the rows: views of one fused product."""
        y = self.ops.lowbit_marlin_gemm(*self.qkv, x, self.hidden, 128).view(x.shape[0], -1, self.head_dim)
        return y.split([self.heads, self.heads_kv, self.heads_kv], dim=1)

    def output(self, a):
        return self.ops.lowbit_marlin_gemm(*self.o, a.view(a.shape[0], -1), self.heads * self.head_dim, 128)

    def prompts(self, x, page_table, seq_lens, cu_seqlens):
        """x [tokens, hidden]: whole prompts, packed; their keys and values enter the cache."""
        q, k, v = self.project(x)
        q, k = self.cache.append(q, k, v, page_table, seq_lens, cu_seqlens, rotation=self.rotation, q_out=q, return_k=True)
        return self.output(prompt_attention(q, k, v, cu_seqlens))

    def step(self, x, page_table, seq_lens):
        """x [batch, hidden]: the next token of every sequence; seq_lens counts it already."""
        q, k, v = self.project(x)
        self.cache.append(q, k, v, page_table, seq_lens, rotation=self.rotation, q_out=q)
        return self.output(self.cache.attend(q, page_table, seq_lens))


def tables(lens, most, page_size, device):
    """Pages handed out in order, enough for `most` tokens a sequence; seq_lens and cu_seqlens of the prompts."""
    per = -(-most // page_size)
    table = torch.arange(len(lens) * per, dtype=torch.int32, device=device).view(len(lens), per)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=device)
    starts = torch.zeros(len(lens) + 1, dtype=torch.int32, device=device)
    starts[1:] = seq_lens.cumsum(0)
    return table, seq_lens, starts


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, nargs="+", default=[300, 41, 1000])
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args(argv)
    most = max(a.prompts) + a.steps
    layer = AttentionLayer(pages=len(a.prompts) * -(-most // 16), positions=most)
    table, lens, starts = tables(a.prompts, most, 16, "cuda")
    x = torch.randn((sum(a.prompts), layer.hidden), device="cuda").half()
    event = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
    for _ in range(2):  # the first to warm up
        layer.prompts(x, table, lens, starts)
        event[0].record()
        y = layer.prompts(x, table, lens, starts)
        event[1].record()
        now = lens.clone()
        for _step in range(a.steps):
            now += 1
            y = layer.step(torch.randn((len(a.prompts), layer.hidden), device="cuda").half(), table, now)
        event[2].record()
        torch.cuda.synchronize()
    print(f"{sum(a.prompts)} prompt tokens: {event[0].elapsed_time(event[1]) * 1e3:.0f} us; "
          f"a step of {len(a.prompts)} tokens: {event[1].elapsed_time(event[2]) * 1e3 / max(1, a.steps):.0f} us; "
          f"output {tuple(y.shape)}, finite: {bool(y.isfinite().all())}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
