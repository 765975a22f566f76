"""The example's attention layer: decoding over the 8-bit cache agrees with prompts of the same tokens, through both projections."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

from tests.gpu_util import print_case

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "attention_layer.py"
    spec = importlib.util.spec_from_file_location("attention_layer_example", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_steps_agree_with_prompts(dev, capsys):
    import torch

    print_case("attention-layer-example")
    E = _example()
    lens, steps = [70, 1, 33], 3
    layer = E.AttentionLayer(hidden=512, heads=8, heads_kv=2, head_dim=64, pages=3 * 5, page_size=16, positions=80, seed=3)
    table, seq_lens, starts = E.tables(lens, 80, 16, dev)
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    rows = [torch.randn((n + steps, 512), device=dev, generator=g).half() for n in lens]
    layer.prompts(torch.cat([r[:n] for r, n in zip(rows, lens)]), table, seq_lens, starts)
    got = []
    for i in range(steps):
        got.append(layer.step(torch.stack([r[n + i] for r, n in zip(rows, lens)]), table, seq_lens + i + 1))
    # the same tokens as whole prompts (the keys and values in fp16 there, in 8 bits above)
    full = [n + steps for n in lens]
    table, seq_lens, starts = E.tables(full, 80, 16, dev)
    want = layer.prompts(torch.cat(rows), table, seq_lens, starts).float()
    spread = float(want.std())
    for i in range(steps):
        for b, n in enumerate(lens):
            row = want[int(starts[b]) + n + i]
            # keys and values rounded to half a step of max / 127, about 1 % of their size, averaged by the softmax
            # and the projection: an output's error is a few per cent of the outputs' spread at most
            assert float((got[i][b].float() - row).abs().max()) < 0.1 * spread, (i, b)
    assert E.main(["--prompts", "40", "3", "--steps", "2"]) == 0
    assert "finite: True" in capsys.readouterr().out
