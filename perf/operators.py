"""The attention between the QKV and the O projection, as cases that can be prepared, run and checked.

Three operators, all fp16 with sums in 32 bits:

* ``append``: the rows of a QKV projection enter a layer's cache.  Queries and
  keys are rotated to their positions (the first ``rot`` values of a head, as
  halves or interleaved pairs); keys and values are stored in 8 bits, pages of
  ``page`` tokens, with one 32-bit scale for each page and head.  A page that
  already holds tokens keeps its scale unless the new ones need a larger one,
  and then its codes are rescaled.
* ``decode``: the few newest tokens of each sequence attend to the sequence's
  pages; heads are grouped, token i of n sees the keys up to its own.
* ``prompt``: causal attention inside each of the packed sequences of a batch
  of prompts, with grouped heads, on keys and values as the projection and the
  rotation leave them.

``listed()`` uses this repository's two attention layouts: 40 query heads on 8
of 128 values (the 5120 -> 7168 QKV projection) and 24 on 4 of 256 (the 14336
wide one, whose other half is the output gate, with 64 rotated values of 256);
``draw`` other heads, pages, batches and lengths of the same ranges.

``own`` chooses between the plain form (elementary torch operations in 32
bits) and the framework's operators.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
F32 = torch.float32


def listed():
    h128 = dict(hq=40, hkv=8, d=128)
    h256 = dict(hq=24, hkv=4, d=256)
    half, inter = dict(rot=64, interleaved=False), dict(rot=128, interleaved=True)
    return [
        # one token of one sequence enters the cache: the smallest call
        {"name": "append_1", "kind": "append", "batch": 1, "new": 1, "lo": 1000, "hi": 1000, "page": 64, "mix": 1, **h256, **half},
        # a decode batch: one token each of 64 sequences
        {"name": "append_64", "kind": "append", "batch": 64, "new": 1, "lo": 20, "hi": 4000, "page": 16, "mix": 2, **h128, **inter},
        # five prompts of different lengths at once
        {"name": "append_prompts", "kind": "append", "batch": 5, "new": 0, "lo": 117, "hi": 2300, "page": 64, "mix": 3, **h256, **half},
        # one long prompt
        {"name": "append_16384", "kind": "append", "batch": 1, "new": 0, "lo": 16384, "hi": 16384, "page": 16, "mix": 4, **h128, **inter},
        # the next token of a short chat: latency
        {"name": "decode_1x301", "kind": "decode", "batch": 1, "new": 1, "lo": 301, "hi": 301, "page": 64, "mix": 5, **h256},
        # three drafted tokens each of five sequences are verified
        {"name": "verify_5x3", "kind": "decode", "batch": 5, "new": 3, "lo": 701, "hi": 6000, "page": 32, "mix": 6, **h128},
        # a full server's decode step over ragged contexts
        {"name": "decode_128", "kind": "decode", "batch": 128, "new": 1, "lo": 500, "hi": 8192, "page": 16, "mix": 7, **h128},
        # one token over a very long document
        {"name": "decode_1x131072", "kind": "decode", "batch": 1, "new": 1, "lo": 131072, "hi": 131072, "page": 64, "mix": 8, **h256},
        # a short question
        {"name": "prompt_97", "kind": "prompt", "batch": 1, "lo": 97, "hi": 97, "mix": 9, **h128},
        # seven prompts packed into one call
        {"name": "prompt_7_packed", "kind": "prompt", "batch": 7, "lo": 100, "hi": 1500, "mix": 10, **h256},
        # long prompts, one sequence each
        {"name": "prompt_8192", "kind": "prompt", "batch": 1, "lo": 8192, "hi": 8192, "mix": 11, **h128},
        {"name": "prompt_16384", "kind": "prompt", "batch": 1, "lo": 16384, "hi": 16384, "mix": 12, **h256},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    while True:
        d = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        case = {"kind": kind, "hq": hq, "hkv": hkv, "d": d, "mix": rng.randrange(1 << 20)}
        if hq > 64 or 3072 in (hq * d, hkv * d):
            continue
        if kind == "append":
            rot = rng.choice([d, d, d // 2, d // 4])
            case.update(page=rng.choice([16, 32, 64, 128]), rot=rot, interleaved=rng.random() < 0.5)
            if rng.random() < 0.5:
                case.update(batch=_log_int(rng, 1, 128), new=rng.choice([1, 1, 1, 2, 3, 4]), lo=_log_int(rng, 8, 500),
                            hi=_log_int(rng, 500, 8192))
            else:
                case.update(batch=_log_int(rng, 1, 16), new=0, lo=1, hi=1)
                case.update(lo=_log_int(rng, 1, 1024), hi=_log_int(rng, 1024, 16384 // case["batch"]))
            fits = sum(_news(case)) * (hq + hkv) * d <= 16384 * 48 * 128
        elif kind == "decode":
            case.update(batch=_log_int(rng, 1, 128), new=rng.choice([1, 1, 2, 3, 4]), page=rng.choice([16, 32, 64, 128]))
            hi = _log_int(rng, 64, 131072)
            case.update(lo=_log_int(rng, 4 + hi // 64, hi), hi=hi)
            fits = case["batch"] * hi * max(hkv * d, 4 * case["new"] * hq) <= 128 * 8192 * 8 * 128
        else:
            hi = _log_int(rng, 16, 16384)
            case.update(batch=_log_int(rng, 1, 16), lo=_log_int(rng, 1 + hi // 64, hi), hi=hi)
            total = sum(_lens(case))
            fits = hq * total * total * max(d, 64) <= 24 * 16384 * 16384 * 256 and hq * total * total <= 24 * 16384 * 16384
        if fits and 3072 not in case.values():
            return case


def _lens(case):
    """The sequences' lengths, spread evenly over their logarithm: the first is the longest."""
    rng = random.Random(case["mix"])
    lo, hi = case["lo"], case["hi"]
    return [hi] + [_log_int(rng, lo, hi) for _ in range(case["batch"] - 1)]


def _news(case):
    """How many tokens of each sequence are new."""
    return [case["new"] or n for n in _lens(case)]


# ------------------------------------------------------------------ inputs ---

def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(counts):
    return _i32([0] + torch.tensor(counts).cumsum(0).tolist())


def _pages(g, counts, pool, width):
    """page_table [batch, width]: `counts[b]` (first, last) pages of the pool in random order, -1 where a sequence has none."""
    order = torch.randperm(pool, device=DEV, generator=g).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, (first, last) in enumerate(counts):
        table[b, first:last] = order[at:at + last - first]
        at += last - first
    return table


def _projected(g, tokens, heads, d):
    """Rows as a QKV projection writes them: a few channels of every head are larger than the rest."""
    x = torch.randn((tokens, heads, d), device=DEV, generator=g)
    return x.mul_(torch.rand((heads, d), device=DEV, generator=g).pow_(8).mul_(4).add_(0.75)).half()


def _codes(g, shape):
    return torch.randn(shape, device=DEV, generator=g, dtype=torch.float16).mul_(36).round_().clamp_(-127, 127).to(torch.int8)


def _scales(g, shape):
    return torch.rand(shape, device=DEV, generator=g).mul_(0.02).add_(0.015)


def _rotation(positions, rot):
    """cos | sin of every position and frequency, base 10000 stretched four times (positions interpolated): float32 [positions, rot]."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] / 4 * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = _lens(case)
    s = {"case": case, "scale": d ** -0.5}
    if case["kind"] == "append":
        news, p = _news(case), case["page"]
        lens = [max(a, b) for a, b in zip(lens, news)]
        tokens = sum(news)
        qkv = _projected(g, tokens, hq + 2 * hkv, d)
        s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], seq_lens=_i32(lens),
                 starts=None if case["new"] else _starts(news))
        touched = [((a - b) // p, (a - 1) // p + 1) for a, b in zip(lens, news)]
        pool = sum(last - first for first, last in touched)
        s["table"] = _pages(g, touched, pool, max(last for _, last in touched))
        # the pages that the call writes, the tokens before the new ones in them
        s.update(k_cache=_codes(g, (pool, hkv, p, d)), v_cache=_codes(g, (pool, hkv, d, p)),
                 k_scale=_scales(g, (pool, hkv)), v_scale=_scales(g, (pool, hkv)))
        held = torch.zeros((pool,), dtype=torch.int64, device=DEV)
        for b, (first, _) in enumerate(touched):
            held[s["table"][b, first].long()] = lens[b] - news[b] - first * p
        empty = torch.arange(p, device=DEV)[None] >= held[:, None]
        s["k_cache"].masked_fill_(empty[:, None, :, None], 0)
        s["v_cache"].masked_fill_(empty[:, None, None, :], 0)
        s["rotation"] = _rotation(max(lens), case["rot"])
        s["q_out"] = torch.empty((tokens, hq, d), dtype=torch.float16, device=DEV)
        s["k_out"] = None if case["new"] else torch.empty((tokens, hkv, d), dtype=torch.float16, device=DEV)
    elif case["kind"] == "decode":
        n, p = case["new"], case["page"]
        lens = [max(a, n) for a in lens]
        counts = [(0, -(-a // p)) for a in lens]
        pool = sum(last for _, last in counts)
        s.update(q=torch.randn((case["batch"] * n, hq, d), device=DEV, generator=g).half(), seq_lens=_i32(lens),
                 table=_pages(g, counts, pool, max(last for _, last in counts)),
                 k_cache=_codes(g, (pool, hkv, p, d)), v_cache=_codes(g, (pool, hkv, d, p)),
                 k_scale=_scales(g, (pool, hkv)), v_scale=_scales(g, (pool, hkv)),
                 out=torch.empty((case["batch"] * n, hq, d), dtype=torch.float16, device=DEV),
                 workspace=torch.zeros((case["batch"] * n * hq,), dtype=torch.int32, device=DEV))
    else:
        tokens = sum(lens)
        qkv = _projected(g, tokens, hq + 2 * hkv, d)
        s.update(q=qkv[:, :hq].contiguous(), k=qkv[:, hq:hq + hkv].contiguous(), v=qkv[:, hq + hkv:], starts=_starts(lens),
                 out=torch.empty((tokens, hq, d), dtype=torch.float16, device=DEV))
    return s


# -------------------------------------------------------- the plain forms ---

def _sequence_of(tokens, starts, batch):
    """For each of the packed tokens: its sequence, its place in it and how many it has."""
    t = torch.arange(tokens, device=DEV)
    if starts is None:
        n = tokens // batch
        return t // n, t % n, n
    b = torch.bucketize(t, starts[1:], right=True)
    return b, t - starts[b], starts[b + 1] - starts[b]


def _rotated(x, cos, sin, interleaved):
    x, half = x.float(), cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _stored(x, cache, scale, page, off, kept):
    """Stores x [tokens, heads, d] at slot `off` of `page`; cache [pages, heads, slots, d] and scale [pages, heads] are updated."""
    pool, heads = scale.shape
    peak = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    written = torch.zeros((pool, 1), dtype=torch.bool, device=DEV)
    older = torch.zeros((pool, 1), dtype=torch.bool, device=DEV)
    written[page, 0] = True
    older[page, 0] = kept
    new = torch.maximum(torch.where(older, scale, torch.zeros_like(scale)), peak * (1.0 / 127))
    new = torch.where(written, new, scale)
    shrink = torch.where(older & (new > scale), scale / new, torch.ones_like(scale))
    cache.copy_((cache.float() * shrink[..., None, None]).round())
    inverse = torch.where(new > 0, new.reciprocal(), torch.zeros_like(new))
    cache[page, :, off] = (x * inverse[page][..., None]).round().clamp(-127, 127).to(torch.int8)
    scale.copy_(new)


def _plain_append(s):
    tokens, p = s["q"].shape[0], s["k_cache"].shape[2]
    b, place, count = _sequence_of(tokens, s["starts"], s["seq_lens"].shape[0])
    start = s["seq_lens"][b] - count
    pos = start + place
    page, off = s["table"][b, pos // p].long(), pos % p
    kept = pos // p * p < start
    half = s["rotation"].shape[1] // 2
    cos, sin = s["rotation"][pos, None, :half], s["rotation"][pos, None, half:]
    q = _rotated(s["q"], cos, sin, s["case"]["interleaved"]).half()
    k = _rotated(s["k"], cos, sin, s["case"]["interleaved"])
    _stored(k, s["k_cache"], s["k_scale"], page, off, kept)
    _stored(s["v"].float(), s["v_cache"].transpose(2, 3), s["v_scale"], page, off, kept)
    return q, None if s["k_out"] is None else k.half()


def _softmax(x):
    """exp(x) over its sum along the last axis; a row of -inf alone gives zeros."""
    peak = x.amax(-1, keepdim=True)
    e = (x - peak.masked_fill(peak == -math.inf, 0)).exp_()
    total = e.sum(-1, keepdim=True)
    return e.div_(total.masked_fill(total == 0, 1))


def _plain_decode(s):
    (rows, hq, d), batch = s["q"].shape, s["seq_lens"].shape[0]
    n, hkv, p = rows // batch, s["k_cache"].shape[1], s["k_cache"].shape[2]
    page = s["table"].clamp(min=0).long()
    wide = page.shape[1] * p
    k = (s["k_cache"][page].float() * s["k_scale"][page][..., None, None]).permute(0, 2, 4, 1, 3).reshape(batch * hkv, d, wide)
    v = (s["v_cache"][page].float() * s["v_scale"][page][..., None, None]).permute(0, 2, 1, 4, 3).reshape(batch * hkv, wide, d)
    q = s["q"].float().reshape(batch, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(batch * hkv, -1, d)
    x = (torch.bmm(q, k) * s["scale"]).view(batch, hkv, n, hq // hkv, wide)
    last = s["seq_lens"][:, None] - n + torch.arange(n, device=DEV)
    hidden = torch.arange(wide, device=DEV) > last[..., None]
    x = _softmax(x.masked_fill_(hidden[:, None, :, None], -math.inf))
    o = torch.bmm(x.view(batch * hkv, -1, wide), v)
    return o.view(batch, hkv, n, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(rows, hq, d).half()


def _plain_prompt(s):
    tokens, hq, d = s["q"].shape
    hkv = s["k"].shape[1]
    b, place, _ = _sequence_of(tokens, s["starts"], 0)
    q = s["q"].float().view(tokens, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
    k, v = s["k"].float().permute(1, 2, 0).contiguous(), s["v"].float().transpose(0, 1).contiguous()
    x = torch.bmm(q, k).mul_(s["scale"]).view(hq, tokens, tokens)
    hidden = (b[:, None] != b) | (place[:, None] < place)
    x = _softmax(x.masked_fill_(hidden, -math.inf))
    o = torch.bmm(x.view(hkv, -1, tokens), v)
    return o.view(hq, tokens, d).transpose(0, 1).half()


# --------------------------------------------------------------------- run ---

def _values(cache, scale):
    """What the codes stand for, in fp16."""
    return torch.mul(cache, scale[..., None, None], out=torch.empty(cache.shape, dtype=torch.float16, device=DEV))


def run(s):
    kind = s["case"]["kind"]
    if own:
        from neurova_amd.ops import cuda_ops
        ops = cuda_ops()
    if kind == "append":
        if own:
            ops.kv8_append_out(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                               s["seq_lens"], s["starts"], s["rotation"], s["q_out"], s["k_out"], s["case"]["interleaved"])
            q, k = s["q_out"], s["k_out"]
        else:
            q, k = _plain_append(s)
        got = {"q": q, "k_cache": _values(s["k_cache"], s["k_scale"]), "v_cache": _values(s["v_cache"], s["v_scale"])}
        return got if k is None else {"k": k, **got}
    if not own:
        return _plain_decode(s) if kind == "decode" else _plain_prompt(s)
    if kind == "decode":
        ops.kv8_attention_out(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["seq_lens"],
                              s["out"], s["workspace"], s["scale"])
    else:
        ops.prompt_attention_out(s["q"], s["k"], s["v"], s["starts"], s["out"], s["scale"])
    return s["out"]


# ---------------------------------------------------------- what it has to do ---

def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = _lens(case)
    if case["kind"] == "append":
        news, p = _news(case), case["page"]
        tokens = sum(news)
        # q, k and v are read, q (and a prompt's k) written rotated, the new codes written; in the pages that
        # hold older tokens those are read and written once more
        b = tokens * d * 2 * (2 * hq + 2 * hkv + (0 if case["new"] else hkv)) + 2 * tokens * hkv * d
        lens = [max(a, n) for a, n in zip(lens, news)]
        older = sum((a - n) % p for a, n in zip(lens, news))
        pages = sum((a - 1) // p + 1 - (a - n) // p for a, n in zip(lens, news))
        # what the program reads of its cache: the values of the written pages
        b += 2 * older * hkv * d * 2 + 2 * pages * hkv * p * d * 3
        return {"bytes": b, "flops": 3 * tokens * (hq + hkv) * case["rot"] + 4 * tokens * hkv * d}
    if case["kind"] == "decode":
        n, p = case["new"], case["page"]
        lens = [max(a, n) for a in lens]
        b = sum(lens) * hkv * d * 2 + sum(-(-a // p) for a in lens) * (8 * hkv + 4) + 2 * case["batch"] * n * hq * d * 2
        return {"bytes": b, "flops": 4.0 * d * hq * sum(n * a - n * (n - 1) // 2 for a in lens)}
    return {"bytes": sum(lens) * d * 2 * (2 * hq + 2 * hkv), "flops": 4.0 * d * hq * sum(a * (a + 1) // 2 for a in lens)}


# ------------------------------------------------------------------- exact ---

def _attended(q, k, v, scale, first):
    """q [n, d] over k, v [m, d] in 64 bits; row i sees the keys up to `first` + i."""
    x = (q @ k.T) * scale
    if first + 1 < k.shape[0]:
        x += torch.full_like(x, -math.inf).triu_(first + 1)
    return torch.softmax(x, dim=-1) @ v


def _exact_append(case, s):
    p, half, g = case["page"], case["rot"] // 2, s["rotation"].double()
    lens, at = s["seq_lens"].tolist(), 0
    values = {n: s[n + "_cache"].double() * s[n + "_scale"].double()[..., None, None] for n in ("k", "v")}
    values["v"] = values["v"].transpose(2, 3)
    spin = {n: s[n].double().clone() for n in ("q", "k")}
    news = _news(case)
    for length, n in zip(lens, news):
        turn = torch.complex(g[length - n:length, None, :half].contiguous(), g[length - n:length, None, half:].contiguous())
        for x in spin.values():
            part = x[at:at + n]
            if case["interleaved"]:
                z = torch.view_as_complex(part[..., :2 * half].reshape(n, -1, half, 2)) * turn
                part[..., :2 * half] = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(part[..., :half].clone(), part[..., half:2 * half].clone()) * turn
                part[..., :half], part[..., half:2 * half] = z.real, z.imag
        at += n
    at = 0
    stored = {"k": spin["k"], "v": s["v"].double()}
    for b, (length, n) in enumerate(zip(lens, news)):
        for page in range((length - n) // p, (length - 1) // p + 1):
            lo, hi = max(length - n, page * p), min(length, (page + 1) * p)
            old, where = lo - page * p, int(s["table"][b, page])
            for name, x in stored.items():
                new = x[at + lo - (length - n):at + hi - (length - n)].transpose(0, 1)
                step = new.abs().amax((1, 2)) / 127
                if old:
                    step = torch.maximum(step, s[name + "_scale"][where].double())
                step = step[:, None, None]
                values[name][where, :, :old] = (values[name][where, :, :old] / step).round() * step
                values[name][where, :, old:old + hi - lo] = (new / step).round().clamp(-127, 127) * step
        at += n
    got = {"q": spin["q"], "k_cache": values["k"], "v_cache": values["v"].transpose(2, 3)}
    return got if case["new"] else {"k": spin["k"], **got}


def exact(case, seed):
    s = prepare(case, seed)
    group = case["hq"] // case["hkv"]
    if case["kind"] == "append":
        return _exact_append(case, s)
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    if case["kind"] == "decode":
        n, p = case["new"], case["page"]
        for b, length in enumerate(s["seq_lens"].tolist()):
            page = s["table"][b, :-(-length // p)].long()
            k = (s["k_cache"][page].double() * s["k_scale"][page].double()[..., None, None]).transpose(0, 1).flatten(1, 2)
            v = (s["v_cache"][page].double() * s["v_scale"][page].double()[..., None, None]).permute(1, 0, 3, 2).flatten(1, 2)
            for h in range(case["hkv"]):
                for j in range(group):
                    o[b * n:(b + 1) * n, h * group + j] = _attended(s["q"][b * n:(b + 1) * n, h * group + j].double(), k[h, :length],
                                                                    v[h, :length], s["scale"], length - n)
        return o
    starts = s["starts"].tolist()
    for lo, hi in zip(starts, starts[1:]):
        for h in range(case["hq"]):
            k, v = s["k"][lo:hi, h // group].double(), s["v"][lo:hi, h // group].double()
            o[lo:hi, h] = _attended(s["q"][lo:hi, h].double(), k, v, s["scale"], 0)
    return o
