"""The operators of a paged key / value cache as timed cases: what a program that decodes with this framework calls for every layer
and step.

  append   new tokens of every sequence into the cache: the packed projection's queries and keys are rotated by their positions,
           keys and values go to their pages
  attend   attention of the new tokens over the cached ones, themselves included: one token a sequence is a decoding step, a few
           are tokens to be verified together, many are a chunk of a prompt behind what is cached already

k_pages, v_pages (pages, page size, kv heads, head dim); page_table (sequences, pages of the longest); lengths (sequences): the tokens
of each with the new ones.  New token i of n sits at place lengths - n + i of its sequence, before place 0 there is none.
`own` = False computes the plain forms in elementary torch operations, True calls the framework."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
BASE = 10000.0
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    gqa = dict(hq=32, hkv=8, hd=128, dtype="bf16")     # the decoding layer of this framework's standing cases
    return [
        # a decoding step of 64 requests that are anywhere between their first token and eight thousand
        dict(name="append_S64_n1", kind="append", S=64, new=1, lo=1, hi=8192, page=16, **gqa),
        # a prompt into an empty cache, its length odd
        dict(name="append_L3001", kind="append", S=1, new=3001, lo=3001, hi=3001, page=64, **gqa),
        # prompts of a training-length batch, one kv head per head; two sequences are shorter and padded on the left
        dict(name="append_S4_L4096_mha", kind="append", S=4, new=4096, lo=2500, hi=4096, page=128, hq=32, hkv=32, hd=128, dtype="bf16"),
        # the fp32 parity configuration, a batch of ragged chunks behind cached content
        dict(name="append_fp32_S4_n331", kind="append", S=4, new=331, lo=300, hi=2048, page=32, hq=8, hkv=8, hd=64, dtype="f32"),
        # the first tokens of a lone short request on one rank's heads: latency
        dict(name="attend_S1_c100", kind="attend", S=1, new=1, lo=100, hi=100, page=16, hq=4, hkv=1, hd=128, dtype="bf16"),
        # the standing decode case, with its cache in pages
        dict(name="attend_S1_c8192", kind="attend", S=1, new=1, lo=8192, hi=8192, page=64, **gqa),
        # a lone request behind a very long context
        dict(name="attend_S1_c131072", kind="attend", S=1, new=1, lo=131072, hi=131072, page=64, **gqa),
        # 64 requests in one step, lengths anywhere
        dict(name="attend_S64_c8192", kind="attend", S=64, new=1, lo=1, hi=8192, page=16, **gqa),
        # one kv head per head, one query row for every key
        dict(name="attend_S16_c4001_mha", kind="attend", S=16, new=1, lo=900, hi=4001, page=128, hq=32, hkv=32, hd=128, dtype="bf16"),
        # the parity configuration
        dict(name="attend_fp32_S3_c2048", kind="attend", S=3, new=1, lo=500, hi=2048, page=32, hq=8, hkv=8, hd=64, dtype="f32"),
        # five tokens of each request verified together, head dim 64
        dict(name="attend_S8_n5_c5000_hd64", kind="attend", S=8, new=5, lo=700, hi=5000, page=32, hq=16, hkv=4, hd=64, dtype="bf16"),
        # a chunk of a long prompt behind eight thousand cached tokens
        dict(name="attend_n512_c8703", kind="attend", S=1, new=512, lo=8703, hi=8703, page=64, **gqa),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["append", "attend", "attend"])
        hkv = rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = dict(kind=kind, page=rng.choice([8, 16, 32, 64, 128, 256]), hkv=hkv, hq=hkv * rng.choice([1, 1, 2, 3, 4, 5, 7, 8]), hd=rng.choice([64, 128, 128]),
                 dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
        if c["hq"] > 64:
            continue
        if kind == "append":
            c["S"] = _log(rng, 1, 96)
            c["new"] = rng.choice([1, _log(rng, 2, 4096)])
            c["hi"] = max(c["new"], _log(rng, 1, 8192))
        else:
            c["S"] = _log(rng, 1, 96)
            c["new"] = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 700)])
            c["hi"] = max(c["new"], _log(rng, 16, 131072))
        c["lo"] = rng.choice([c["hi"], rng.randint(0, c["hi"]), rng.randint(0, 1)])
        w, item = work(c), 2 if c["dtype"] == "bf16" else 4
        cache = 2 * c["S"] * c["hi"] * hkv * c["hd"]
        scores = c["S"] * c["hq"] * c["new"] * c["hi"] if kind == "attend" else 0
        if c["lo"] == c["hi"] == 0 or sum(_lengths(c)) == 0:
            continue
        if kind == "append" and w["bytes"] > 0.75e9 or kind == "attend" and (w["bytes"] > 1.0e9 or w["flops"] > 6.5e10):
            continue
        if cache * item <= 2.2e9 and scores <= 1.5e8:
            return c


def _lengths(c):
    """One length per sequence, spread evenly from lo to hi in a scattered order; the first is hi."""
    return [c["hi"] - int((c["hi"] - c["lo"]) * ((i * 0.6180339887498949) % 1.0) + 0.5) for i in range(c["S"])]


def _present(c):
    """New tokens of all sequences that exist."""
    return sum(min(n, c["new"]) for n in _lengths(c))


def work(c):
    item = 2 if c["dtype"] == "bf16" else 4
    tokens, heads = _present(c), c["hq"] + 2 * c["hkv"]
    small = 4 * c["S"] + 4 * sum((n + c["page"] - 1) // c["page"] for n in _lengths(c))
    if c["kind"] == "append":
        return dict(bytes=2 * tokens * heads * c["hd"] * item + small, flops=3 * tokens * (c["hq"] + c["hkv"]) * c["hd"])
    pairs = 0
    for n in _lengths(c):
        m = min(n, c["new"])
        pairs += m * n - m * (m - 1) // 2
    keys = sum(_lengths(c))
    rows = c["S"] * c["new"] * c["hq"]
    return dict(bytes=2 * keys * c["hkv"] * c["hd"] * item + 2 * rows * c["hd"] * item + 4 * rows + small, flops=4 * c["hq"] * c["hd"] * pairs)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[c["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)  # noqa: E731
    s = SimpleNamespace(case=c)
    lengths = _lengths(c)
    s.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    used = [(n + c["page"] - 1) // c["page"] for n in lengths]
    pages = sum(used) + 3                                     # a few that belong to nobody
    order = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    column = torch.arange(max(used), device=DEV)[None, :]
    count = torch.tensor(used, device=DEV)[:, None]
    first = torch.cumsum(count, 0) - count
    s.page_table = torch.where(column < count, order[(first + column).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=DEV)).contiguous()
    shape = (pages, c["page"], c["hkv"], c["hd"])
    s.k_pages, s.v_pages = torch.empty(shape, dtype=dt, device=DEV), torch.empty(shape, dtype=dt, device=DEV)
    for t in (s.k_pages, s.v_pages):
        t.normal_(generator=g)
    if c["kind"] == "append":
        s.qkv = normal(c["S"], c["new"], c["hq"] + 2 * c["hkv"], c["hd"])
        s.inv_freq = (1.0 / (BASE ** (torch.arange(0, c["hd"], 2, dtype=torch.int64).float() / c["hd"]))).to(DEV)   # on the host, as rotary modules do
    else:
        s.q = normal(c["S"], c["new"], c["hq"], c["hd"])
    return s


def run(s):
    c = s.case
    if own:
        from odysseus_transformer_amd import ops
        if c["kind"] == "append":
            q = ops.paged_append_(s.qkv, c["hq"], s.k_pages, s.v_pages, s.page_table, s.lengths, inv_freq=s.inv_freq)
            return q, s.k_pages, s.v_pages
        return ops.paged_attn(s.q, s.k_pages, s.v_pages, s.page_table, s.lengths)
    return _append(s) if c["kind"] == "append" else _attend(s)


def _places(s):
    """(S, n): where the new tokens sit in their sequences, negative: nowhere."""
    n = s.case["new"]
    return s.lengths.long()[:, None] - n + torch.arange(n, device=DEV)[None, :]


def _append(s):
    c = s.case
    place, half = _places(s), c["hd"] // 2
    there = place >= 0
    # the angle is the 32-bit product of position and frequency, cosine and sine are rounded to the values' type: as the framework's
    # and the host model's rotary embedding have them
    angle = (place.float()[:, :, None] * s.inv_freq).double()
    cos, sin = (f(angle).to(s.qkv.dtype).float()[:, :, None, :] for f in (torch.cos, torch.sin))
    x = s.qkv[:, :, :c["hq"] + c["hkv"]].float()
    a, b = x[..., :half], x[..., half:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(s.qkv.dtype)
    q = torch.where(there[:, :, None, None], turned[:, :, :c["hq"]], torch.zeros((), dtype=s.qkv.dtype, device=DEV))
    page = s.page_table.long().gather(1, place.clamp(min=0) // c["page"])
    page, row = page[there], place[there] % c["page"]
    s.k_pages[page, row] = turned[:, :, c["hq"]:][there]
    s.v_pages[page, row] = s.qkv[:, :, c["hq"] + c["hkv"]:][there]
    return q, s.k_pages, s.v_pages


def _attend(s):
    c = s.case
    S, n, hq, hkv, hd = c["S"], c["new"], c["hq"], c["hkv"], c["hd"]
    group = hq // hkv
    page = s.page_table.long().clamp(min=0)
    keys, values = (t[page].flatten(1, 2).float().transpose(1, 2) for t in (s.k_pages, s.v_pages))          # (S, Hkv, keys, D)
    q = s.q.float().view(S, n, hkv, group, hd).permute(0, 2, 3, 1, 4).reshape(S, hkv, group * n, hd)
    scores = torch.matmul(q, keys.transpose(2, 3)).view(S, hkv, group, n, -1) * (1.0 / math.sqrt(hd))
    seen = torch.arange(scores.shape[-1], device=DEV)[None, None, :] <= _places(s)[:, :, None]              # (S, n, keys)
    scores = torch.where(seen[:, None, None], scores, torch.full((), -math.inf, device=DEV))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(S, hkv, group * n, -1), values).view(S, hkv, group, n, hd) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (torch.log(total) + top).squeeze(-1).reshape(S, hq, n)
    return out.permute(0, 3, 1, 2, 4).reshape(S, n, hq, hd).to(s.q.dtype), lse


def exact(c, seed):
    s = prepare(c, seed)
    n, hq, hkv, hd, page = c["new"], c["hq"], c["hkv"], c["hd"], c["page"]
    lengths, table = _lengths(c), s.page_table.tolist()
    if c["kind"] == "append":
        q = torch.zeros((c["S"], n, hq, hd), dtype=torch.float64, device=DEV)
        k_pages, v_pages = s.k_pages.double(), s.v_pages.double()
        # the angle in 32 bits is part of the definition, as the rounding of cosine and sine is
        for b, length in enumerate(lengths):
            m = min(n, length)
            if m == 0:
                continue
            at = torch.arange(length - m, length, device=DEV)
            th = torch.outer(at.float(), s.inv_freq).double()
            turn = torch.complex(torch.cos(th).to(s.qkv.dtype).double(), torch.sin(th).to(s.qkv.dtype).double())[:, None, :]
            new = s.qkv[b, n - m:].double()
            z = torch.complex(new[:, :hq + hkv, :hd // 2].contiguous(), new[:, :hq + hkv, hd // 2:].contiguous()) * turn
            rotated = torch.cat((z.real, z.imag), -1)
            q[b, n - m:] = rotated[:, :hq]
            rows = torch.tensor(table[b], device=DEV)[at // page] * page + at % page
            k_pages.view(-1, hkv, hd)[rows] = rotated[:, hq:]
            v_pages.view(-1, hkv, hd)[rows] = new[:, hq + hkv:]
        return q, k_pages, v_pages
    out = torch.zeros((c["S"], n, hq, hd), dtype=torch.float64, device=DEV)
    lse = torch.full((c["S"], hq, n), -math.inf, dtype=torch.float64, device=DEV)
    for b, length in enumerate(lengths):
        m = min(n, length)
        if m == 0:
            continue
        ids = torch.tensor(table[b][:(length + page - 1) // page], device=DEV)
        k, v = (t[ids].reshape(-1, hkv, hd)[:length].double() for t in (s.k_pages, s.v_pages))
        future = torch.ones((m, length), dtype=torch.bool, device=DEV).triu(length - m + 1)
        for h in range(hq):
            x = (s.q[b, n - m:, h].double() @ k[:, h * hkv // hq].t() / math.sqrt(hd)).masked_fill(future, -math.inf)
            lse[b, h, n - m:] = torch.logsumexp(x, -1)
            out[b, n - m:, h] = torch.softmax(x, -1) @ v[:, h * hkv // hq]
    return out, lse
