"""The operators of decoding over a paged key / value cache in 8 bits, and of choosing the next tokens, as timed cases.

  append   new tokens of every sequence into the cache: queries and keys of the packed projection are rotated by their positions, keys and values are
           stored as e4m3 values with a power of two for each block of tokens and head; what the cache holds then is read back
  read     the values of a cache, gathered by the page table: what a program takes to another cache or looks at
  attend   attention of the new tokens over the cached ones, themselves included
  sample   a token of each row of logits by temperature, top-k, top-p and min-p from a given random number, and its log-probability

k_pages, v_pages (pages, page size, kv heads, head dim) e4m3; k_scales, v_scales (pages, page size / block, kv heads) e8m0; page_table (sequences, pages of
the longest); lengths (sequences): the tokens of each with the new ones.  New token i of n sits at place lengths - n + i of its sequence, before place 0
there is none.  The scale of a block is the least power of two 2^e, e from -126 on, with max |x| <= 448 * 2^e over the finite values of its tokens and
head; where the block holds earlier tokens it is at least what it was, and they are rounded to the new one.

sample orders a row's tokens by falling logits, the lower index first among equals, with weights exp((logit - largest) / temperature).  The first of them is kept
always; the others while they are among the first top_k (0: all), the weights before them are less than top_p times those of all that top_k keeps (1: all), and their
own is at least min_p.  The token is the first whose weights up to and with it exceed the random number times those of all that is kept.  Temperature 0: the first.
`own` = False computes the plain forms in elementary torch operations, True calls the framework."""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
BASE = 10000.0
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def listed():
    gqa = dict(hq=32, hkv=8, hd=128, dtype="bf16")     # the decoding layer of this framework's standing cases
    return [
        # a decoding step of 64 requests early in their answers
        dict(name="append_S64_n1", kind="append", S=64, new=1, lo=1, hi=128, page=64, block=32, **gqa),
        # prompts of a training-length batch, one kv head per head; two sequences are shorter and padded on the left
        dict(name="append_S4_L4096_mha", kind="append", S=4, new=4096, lo=2500, hi=4096, page=128, block=64, hq=32, hkv=32, hd=128, dtype="bf16"),
        # the fp32 parity configuration, a batch of ragged chunks behind cached content
        dict(name="append_fp32_S4_n331", kind="append", S=4, new=331, lo=300, hi=2048, page=32, block=16, hq=8, hkv=8, hd=64, dtype="f32"),
        # a finished prompt is handed to another cache
        dict(name="read_S1_c8191", kind="read", S=1, new=1, lo=8191, hi=8191, page=64, block=32, **gqa),
        # the caches of a ragged batch
        dict(name="read_S16_c4001_hd64", kind="read", S=16, new=1, lo=0, hi=4001, page=16, block=8, hq=16, hkv=16, hd=64, dtype="bf16"),
        # one request: a decoding step's attention, where few rows have to keep the whole card busy
        dict(name="attend_S1_c8192", kind="attend", S=1, new=1, lo=8192, hi=8192, page=64, block=32, **gqa),
        # 64 requests in one step, lengths anywhere
        dict(name="attend_S64_c8192", kind="attend", S=64, new=1, lo=1, hi=8192, page=64, block=32, **gqa),
        # five tokens of each request verified together, head dim 64
        dict(name="attend_S8_n5_c5000_hd64", kind="attend", S=8, new=5, lo=700, hi=5000, page=32, block=16, hq=16, hkv=4, hd=64, dtype="bf16"),
        # a chunk of a long prompt behind eight thousand cached tokens
        dict(name="attend_n512_c8703", kind="attend", S=1, new=512, lo=8703, hi=8703, page=64, block=64, **gqa),
        # the next token of a lone request: latency
        dict(name="sample_R1_V32000", kind="sample", rows=1, vocab=32000, dtype="bf16", temperature=0.8, top_k=0, top_p=0.95, min_p=0.0, mixed=False, masked=False),
        # a serving batch in which every request has its own settings, some with most of their tokens forbidden
        dict(name="sample_R64_V32001_mixed", kind="sample", rows=64, vocab=32001, dtype="f32", temperature=1.0, top_k=50, top_p=0.9, min_p=0.02, mixed=True, masked=True),
        # many samples over a large vocabulary, nothing cut off
        dict(name="sample_R256_V128000", kind="sample", rows=256, vocab=128000, dtype="bf16", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, masked=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["append", "read", "attend", "attend", "sample", "sample"])
        if kind == "sample":
            c = dict(kind=kind, rows=_log(rng, 1, 512), vocab=_log(rng, 500, 262144), dtype=rng.choice(["bf16", "f32"]),
                     temperature=rng.choice([1.0, round(rng.uniform(0.3, 1.5), 2)]), top_k=rng.choice([0, 0, 1, 20, 50, _log(rng, 2, 4000)]),
                     top_p=rng.choice([1.0, 0.95, round(rng.uniform(0.1, 1.0), 3)]), min_p=rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.0, 0.3), 3)]),
                     mixed=rng.choice([False, True]), masked=rng.choice([False, False, True]))
            if c["rows"] * c["vocab"] <= 256 * 128000:
                return c
            continue
        hkv = rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = dict(kind=kind, page=rng.choice([8, 16, 32, 64, 128, 256]), hkv=hkv, hq=hkv * rng.choice([1, 1, 2, 3, 4, 5, 7, 8]), hd=rng.choice([64, 128, 128]),
                 dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
        c["block"] = rng.choice([b for b in (8, 16, 32, 64) if b <= c["page"]])
        if c["hq"] > 64:
            continue
        c["S"] = _log(rng, 1, 96)
        if kind == "append":
            c["new"] = rng.choice([1, _log(rng, 2, 4096)])
            c["hi"] = max(c["new"], _log(rng, 1, 8192))
        elif kind == "read":
            c["new"] = 1
            c["hi"] = _log(rng, 16, 16384)
        else:
            c["new"] = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 700)])
            c["hi"] = max(c["new"], _log(rng, 16, 131072))
        c["lo"] = rng.choice([c["hi"], rng.randint(0, c["hi"]), rng.randint(0, 1)])
        if sum(_lengths(c)) == 0:
            continue
        w = work(c)
        cache = c["S"] * c["hi"] * c["hkv"] * c["hd"]
        scores = c["S"] * c["hq"] * c["new"] * c["hi"] if kind == "attend" else 0
        if w["bytes"] <= (0.5e9 if kind == "attend" else 0.9e9) and w["flops"] <= 7.0e10 and cache <= 3.0e8 and scores <= 1.5e8:
            return c


def _lengths(c):
    """One length per sequence, spread evenly from lo to hi in a scattered order; the first is hi."""
    return [c["hi"] - int((c["hi"] - c["lo"]) * ((i * 0.6180339887498949) % 1.0) + 0.5) for i in range(c["S"])]


def _present(c):
    """New tokens of all sequences that exist."""
    return sum(min(n, c["new"]) for n in _lengths(c))


def work(c):
    if c["kind"] == "sample":
        item = 2 if c["dtype"] == "bf16" else 4
        return dict(bytes=c["rows"] * (c["vocab"] * item + (32 if c["mixed"] else 16)), flops=10 * c["rows"] * c["vocab"])
    item = 2 if c["dtype"] == "bf16" else 4
    lengths, row = _lengths(c), c["hkv"] * c["hd"]
    keys = sum(lengths)
    small = 4 * c["S"] + 4 * sum((n + c["page"] - 1) // c["page"] for n in lengths)
    scales = 2 * c["hkv"] * sum((n + c["block"] - 1) // c["block"] for n in lengths)
    if c["kind"] == "read":
        return dict(bytes=2 * keys * row + scales + small + 2 * 2 * c["S"] * c["hi"] * row, flops=2 * keys * row)
    if c["kind"] == "append":
        tokens = _present(c)
        # the projection in, queries and the new rows out; the values that the cache holds then: its rows in, 16 bits a value out
        return dict(bytes=tokens * (c["hq"] + 2 * c["hkv"]) * c["hd"] * item + c["S"] * c["new"] * c["hq"] * c["hd"] * item + 2 * tokens * row + 2 * keys * row
                    + 2 * 2 * c["S"] * c["hi"] * row + 2 * scales + small, flops=tokens * (3 * c["hq"] + 6 * c["hkv"]) * c["hd"])
    pairs = 0
    for n in lengths:
        m = min(n, c["new"])
        pairs += m * n - m * (m - 1) // 2
    rows = c["S"] * c["new"] * c["hq"]
    return dict(bytes=2 * keys * row + scales + 2 * rows * c["hd"] * item + 4 * rows + small, flops=4 * c["hq"] * c["hd"] * pairs)


# ------------------------------------------------------------------ inputs
def _exponent(top):
    """The least e from -126 on with top <= 448 * 2^e, of 32-bit values."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 8 - (m <= 0.875).to(x.dtype), torch.full_like(x, -126)).clamp(-126, 127)


def _filled(shape, block, g):
    """Pages as a program finds them: keys (or values) of unit size, some channels larger, in their blocks' scales.  Heads lie outside of rows, as the framework's
    cache has them."""
    pages, page, hkv, hd = shape
    values = torch.empty((pages, hkv, page, hd), dtype=F8, device=DEV)
    scales = torch.empty((pages, hkv, page // block), dtype=E8, device=DEV)
    channel = torch.exp(0.5 * torch.randn((hkv, 1, 1, hd), generator=g, device=DEV))
    step = max(1, (1 << 25) // (page * hkv * hd))
    for p in range(0, pages, step):
        x = torch.randn((min(step, pages - p), hkv, page // block, block, hd), generator=g, device=DEV) * channel
        e = _exponent(x.abs().amax((-1, -2)))
        values[p:p + step] = torch.ldexp(x, -e[..., None, None]).to(F8).flatten(2, 3)
        scales[p:p + step] = (e + 127).to(torch.uint8).view(E8)
    return values.transpose(1, 2), scales.transpose(1, 2)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = SimpleNamespace(case=c)
    if c["kind"] == "sample":
        rows, vocab = c["rows"], c["vocab"]
        # a language model's logits: a wide bell, and a few tokens that the context speaks for
        s.logits = 2.0 * torch.randn((rows, vocab), generator=g, device=DEV)
        likely = torch.randint(0, vocab, (rows, 24), generator=g, device=DEV)
        s.logits.scatter_add_(1, likely, 12.0 * torch.rand((rows, 24), generator=g, device=DEV))
        if c["masked"]:   # every third row may only answer with a few of its tokens
            forbidden = torch.rand((rows, vocab), generator=g, device=DEV) < 0.99
            forbidden[torch.arange(rows, device=DEV) % 3 != 0] = False
            forbidden.scatter_(1, likely, False)
            s.logits.masked_fill_(forbidden, -math.inf)
        s.logits = s.logits.to(TYPES[c["dtype"]])
        s.u = torch.rand((rows,), generator=g, device=DEV)
        s.temperature, s.top_k, s.top_p, s.min_p = c["temperature"], c["top_k"], c["top_p"], c["min_p"]
        if c["mixed"]:    # each row its own: some greedy, some without one cut or the other
            some = torch.rand((4, rows), generator=g, device=DEV)
            s.temperature = torch.where(some[0] < 0.1, 0.0, s.temperature * (0.5 + some[0]))
            s.top_k = torch.where(some[1] < 0.3, 0, torch.ceil(s.top_k * 2 * some[1])).to(torch.int32)
            s.top_p = torch.where(some[2] < 0.3, 1.0, s.top_p * (0.5 + 0.5 * some[2]))
            s.min_p = torch.where(some[3] < 0.3, 0.0, s.min_p * some[3])
        return s
    dt = TYPES[c["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)  # noqa: E731
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
    (s.k_pages, s.k_scales), (s.v_pages, s.v_scales) = _filled(shape, c["block"], g), _filled(shape, c["block"], g)
    if c["kind"] == "append":
        s.qkv = normal(c["S"], c["new"], c["hq"] + 2 * c["hkv"], c["hd"])
        s.inv_freq = (1.0 / (BASE ** (torch.arange(0, c["hd"], 2, dtype=torch.int64).float() / c["hd"]))).to(DEV)   # on the host, as rotary modules do
    elif c["kind"] == "attend":
        s.q = normal(c["S"], c["new"], c["hq"], c["hd"])
    return s


def run(s):
    c = s.case
    if own:
        from odysseus_transformer_amd import ops
        if c["kind"] == "sample":
            return ops.sample(s.logits, s.u, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)
        cache = (s.k_pages, s.v_pages, s.k_scales, s.v_scales, s.page_table, s.lengths)
        if c["kind"] == "append":
            q = ops.paged_append_q8_(s.qkv, c["hq"], *cache, inv_freq=s.inv_freq)
            return (q, *ops.paged_read_q8(*cache, c["hi"]))
        if c["kind"] == "read":
            return ops.paged_read_q8(*cache, c["hi"])
        return ops.paged_attn_q8(s.q, *cache)
    if c["kind"] == "sample":
        return _sample(s)
    if c["kind"] == "append":
        return (_append(s), *_read(s, torch.bfloat16))
    return _read(s, torch.bfloat16) if c["kind"] == "read" else _attend(s)


# ------------------------------------------------------------------ the plain forms
def _places(s):
    """(S, n): where the new tokens sit in their sequences, negative: nowhere."""
    n = s.case["new"]
    return s.lengths.long()[:, None] - n + torch.arange(n, device=DEV)[None, :]


def _rows(s, place):
    """Pages and rows of places, and which of them there are."""
    c = s.case
    there = (place >= 0) & (place < s.lengths.long()[:, None])
    page = s.page_table.long().gather(1, (place.clamp(min=0) // c["page"]).clamp(max=s.page_table.shape[1] - 1))
    return page.clamp(min=0), place % c["page"], there & (page >= 0)


def _store(s, pages, scales, new):
    """The new tokens' rows (S, n, Hkv, D), in 32 bits, to their places."""
    c = s.case
    n, b, hkv, hd = c["new"], c["block"], c["hkv"], c["hd"]
    blocks = (n + b - 2) // b + 1
    first = s.lengths.long()[:, None] - n                                                     # of the new tokens
    start = torch.div(first.clamp(min=0), b, rounding_mode="floor") * b                       # of the blocks that they reach
    place = start + torch.arange(blocks * b, device=DEV)[None, :]
    page, row, there = _rows(s, place)
    fresh = there & (place >= first)
    shape = (c["S"], blocks, b, hkv, hd)
    x = new.gather(1, (place - first).clamp(0, n - 1)[:, :, None, None].expand(-1, -1, hkv, hd)).view(shape)
    mine = fresh.view(c["S"], blocks, b, 1, 1)
    top = torch.where(mine & torch.isfinite(x), x.abs(), torch.zeros((), device=DEV)).amax((2, 4))                                  # (S, blocks, Hkv)
    at, has_old = place.view(c["S"], blocks, b)[:, :, 0], (there & ~fresh).view(c["S"], blocks, b).any(2)
    of_block, line = page.view(c["S"], blocks, b)[:, :, 0], at % c["page"] // b
    before = scales.view(torch.uint8)[of_block, line].int() - 127
    e = _exponent(top)
    e = torch.where(has_old[:, :, None], torch.maximum(e, before), e)
    old = torch.ldexp(pages[page, row].view(shape).float(), (before - e)[:, :, None, :, None])
    held = torch.where(mine, torch.ldexp(x, -e[:, :, None, :, None]), old).to(F8).flatten(1, 2)
    pages.view(torch.uint8)[page[there], row[there]] = held.view(torch.uint8)[there]
    touched = fresh.view(c["S"], blocks, b).any(2)
    scales.view(torch.uint8)[of_block[touched], line[touched]] = (e + 127).to(torch.uint8)[touched]


def _append(s):
    c = s.case
    place, half = _places(s), c["hd"] // 2
    # the angle is the 32-bit product of position and frequency, cosine and sine are rounded to the values' type: as the framework's
    # and the host model's rotary embedding have them
    angle = (place.float()[:, :, None] * s.inv_freq).double()
    cos, sin = (f(angle).to(s.qkv.dtype).double()[:, :, None, :] for f in (torch.cos, torch.sin))
    # 64 bits until a value is rounded to the eight that the cache holds: next to a border 32 would choose the other one now and then
    x = s.qkv[:, :, :c["hq"] + c["hkv"]].double()
    a, b = x[..., :half], x[..., half:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    q = torch.where((place >= 0)[:, :, None, None], turned[:, :, :c["hq"]].to(s.qkv.dtype), torch.zeros((), dtype=s.qkv.dtype, device=DEV))
    _store(s, s.k_pages, s.k_scales, turned[:, :, c["hq"]:].float())
    _store(s, s.v_pages, s.v_scales, s.qkv[:, :, c["hq"] + c["hkv"]:].float())
    return q


def _read(s, dtype):
    c = s.case
    place = torch.arange(c["hi"], device=DEV)[None, :].expand(c["S"], -1)
    page, row, there = _rows(s, place)
    line, there = row // c["block"], there[:, :, None, None]
    return tuple(torch.where(there, pages[page, row].float() * scales[page, line].float()[..., None], torch.zeros((), device=DEV)).to(dtype)
                 for pages, scales in ((s.k_pages, s.k_scales), (s.v_pages, s.v_scales)))


def _attend(s):
    c = s.case
    S, n, hq, hkv, hd = c["S"], c["new"], c["hq"], c["hkv"], c["hd"]
    group = hq // hkv
    keys, values = (t.transpose(1, 2).contiguous() for t in _read(s, torch.float32))                        # (S, Hkv, keys, D)
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


def _column(v, dtype):
    """A setting of each row, or one for all."""
    return v.to(dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((1, 1), v, dtype=dtype, device=DEV)


def _sample(s):
    # in 64 bits: sums of many weights are compared with one another
    t, k, p, m = _column(s.temperature, torch.float64), _column(s.top_k, torch.int64), _column(s.top_p, torch.float64), _column(s.min_p, torch.float64)
    x, index = torch.sort(s.logits.double(), dim=-1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=DEV)[None, :]
    one = rank == 0
    d = torch.where(t > 0, (x - x[:, :1]) / t, torch.where(one, 0.0, -math.inf).double())
    w = torch.exp(d)
    w = torch.where((rank < k) | (k <= 0), w, torch.zeros_like(w))
    upto = torch.cumsum(w, -1)
    keep = one | (((upto - w < p * upto[:, -1:]) | (p >= 1)) & (w >= m) & (w > 0))
    w = torch.where(keep, w, torch.zeros_like(w))
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    at = (upto <= s.u.double()[:, None] * total).sum(-1, keepdim=True)
    at = torch.minimum(at, keep.sum(-1, keepdim=True) - 1)
    return index.gather(1, at)[:, 0], (d.gather(1, at) - torch.log(total))[:, 0].float()


# ------------------------------------------------------------------ the definitions in 64 bits
def _e4m3(x):
    """x, at most 448, to the nearest value of four bits of mantissa and exponents from -6 on, half way to the even one."""
    step = torch.exp2((torch.frexp(x)[1].double() - 1).clamp(min=-6.0) - 3.0)
    return torch.round(x / step) * step


def _held(s, pages, scales, sequence, length):
    """What the cache holds of a sequence: (length, Hkv, D), and the exponents of its blocks."""
    c = s.case
    ids = s.page_table[sequence, :(length + c["page"] - 1) // c["page"]].long()
    e = scales.view(torch.uint8)[ids].flatten(0, 1).double() - 127
    return pages[ids].flatten(0, 1).double()[:length] * torch.exp2(e).repeat_interleave(c["block"], 0)[:length, :, None], e


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "sample":
        return _exact_sample(s)
    n, hq, hkv, hd, b = c["new"], c["hq"], c["hkv"], c["hd"], c["block"]
    lengths = _lengths(c)
    if c["kind"] == "attend":
        out = torch.zeros((c["S"], n, hq, hd), dtype=torch.float64, device=DEV)
        lse = torch.full((c["S"], hq, n), -math.inf, dtype=torch.float64, device=DEV)
        for i, length in enumerate(lengths):
            m = min(n, length)
            if m == 0:
                continue
            k, v = _held(s, s.k_pages, s.k_scales, i, length)[0], _held(s, s.v_pages, s.v_scales, i, length)[0]
            future = torch.ones((m, length), dtype=torch.bool, device=DEV).triu(length - m + 1)
            for h in range(hq):
                x = (s.q[i, n - m:, h].double() @ k[:, h * hkv // hq].t() / math.sqrt(hd)).masked_fill(future, -math.inf)
                lse[i, h, n - m:] = torch.logsumexp(x, -1)
                out[i, n - m:, h] = torch.softmax(x, -1) @ v[:, h * hkv // hq]
        return out, lse
    held = [torch.zeros((c["S"], c["hi"], hkv, hd), dtype=torch.float64, device=DEV) for _ in range(2)]
    if c["kind"] == "read":
        for i, length in enumerate(lengths):
            for to, pages, scales in zip(held, (s.k_pages, s.v_pages), (s.k_scales, s.v_scales)):
                if length:
                    to[i, :length] = _held(s, pages, scales, i, length)[0]
        return tuple(held)
    q = torch.zeros((c["S"], n, hq, hd), dtype=torch.float64, device=DEV)
    for i, length in enumerate(lengths):
        m = min(n, length)
        if m == 0:
            continue
        at = torch.arange(length - m, length, device=DEV)
        # the angle in 32 bits is part of the definition, as the rounding of cosine and sine is
        th = torch.outer(at.float(), s.inv_freq).double()
        turn = torch.complex(torch.cos(th).to(s.qkv.dtype).double(), torch.sin(th).to(s.qkv.dtype).double())[:, None, :]
        x = s.qkv[i, n - m:].double()
        z = torch.complex(x[:, :hq + hkv, :hd // 2].contiguous(), x[:, :hq + hkv, hd // 2:].contiguous()) * turn
        turned = torch.cat((z.real, z.imag), -1)
        q[i, n - m:] = turned[:, :hq]
        for to, pages, scales, new in ((held[0], s.k_pages, s.k_scales, turned[:, hq:]), (held[1], s.v_pages, s.v_scales, x[:, hq + hkv:])):
            whole, e = _held(s, pages, scales, i, length)
            whole[length - m:] = new
            for j in range((length - m) // b, (length + b - 1) // b):
                block, since = slice(j * b, min(j * b + b, length)), max(length - m, j * b)
                top = whole[since:block.stop].abs().amax((0, 2))
                new_e = torch.ceil(torch.log2((top / 448.0).clamp(min=2.0 ** -126)))
                new_e = torch.where(torch.exp2(new_e - 1) * 448.0 >= top, new_e - 1, new_e).clamp(min=-126.0)
                if since > j * b:
                    new_e = torch.maximum(new_e, e[j])
                factor = torch.exp2(new_e)[None, :, None]
                whole[block] = _e4m3(whole[block] / factor) * factor
            to[i, :length] = whole
    return q, held[0], held[1]


def _exact_sample(s):
    rows, vocab = s.logits.shape
    of = lambda v, r: float(v[r]) if isinstance(v, torch.Tensor) else float(v)  # noqa: E731
    tokens, logs = [], []
    for r in range(rows):
        x = s.logits[r].double()
        t, k, p, m = (of(v, r) for v in (s.temperature, s.top_k, s.top_p, s.min_p))
        order = torch.sort(-x, stable=True)[1]
        if t == 0:
            tokens.append(order[0])
            logs.append(torch.zeros((), dtype=torch.float64, device=DEV))
            continue
        w = torch.exp((x[order] - x.max()) / t)
        kept = w[:int(k)] if k > 0 else w
        sums = torch.cumsum(kept, 0)
        if p < 1:
            kept = kept[:max(1, int((sums[:-1] < p * sums[-1]).sum()) + 1)]
        kept = kept[:max(1, int((kept >= m).sum()))]
        kept = kept[kept > 0]
        sums = torch.cumsum(kept, 0)
        at = min(int(torch.searchsorted(sums, s.u[r].double() * sums[-1], right=True)), len(kept) - 1)
        tokens.append(order[at])
        logs.append(torch.log(kept[at] / sums[-1]))
    return torch.stack(tokens), torch.stack(logs)
