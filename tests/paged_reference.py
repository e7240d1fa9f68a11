"""A key / value cache in pages in 64 bits on the CPU: what tests compare the kernels with."""
import math

import torch


def make(lengths, n, Hq, Hkv, D, page, dtype, seed, spare=3, layout="rows"):
    """Random content, pages in a scattered order: dict of CPU tensors.  layout: 'rows' (pages, page, Hkv, D), 'heads' (pages, Hkv, page, D)
    seen as rows, 'mixed': one pool (pages, 2, page, Hkv, D) with a wider row of heads."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g).to(dtype)  # noqa: E731
    S = len(lengths)
    used = [(max(x, 0) + page - 1) // page for x in lengths]
    pages, width = sum(used) + spare, max(used + [1]) + 1
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((S, width), -1, dtype=torch.int32)
    for s in range(S):
        for c in range(used[s]):
            table[s, c] = order.pop()
    if layout == "rows":
        k, v = normal(pages, page, Hkv, D), normal(pages, page, Hkv, D)
    elif layout == "heads":
        k, v = normal(pages, Hkv, page, D).transpose(1, 2), normal(pages, Hkv, page, D).transpose(1, 2)
    else:
        pool = normal(pages, 2, page, Hkv + 1, D)
        k, v = pool[:, 0, :, :Hkv], pool[:, 1, :, 1:]
    return dict(k=k, v=v, table=table, lengths=torch.tensor(lengths, dtype=torch.int32), qkv=normal(S, n, Hq + 2 * Hkv, D), q=normal(S, n, Hq, D),
                page=page)


def page_of(c, s, place):
    """(page, row) of a place, None where it has none."""
    column = place // c["page"]
    if place < 0 or column >= c["table"].shape[1]:
        return None
    p = int(c["table"][s, column])
    return (p, place % c["page"]) if 0 <= p < c["k"].shape[0] else None


def first_token(c, s, n):
    """The first of a sequence's n rows that is a token, n if none is: c["new"], where it is there, numbers them."""
    length = max(int(c["lengths"][s]), 0)
    new = n if c.get("new") is None else min(max(int(c["new"][s]), 0), n)
    return max(n - new, min(n - length, n))


def append(c, Hq, inv_freq=None, positions=None):
    """-> q, k_pages, v_pages in float64 (copies), and for each an array of |a cos| + |b sin|, the scale of the products in it."""
    x = c["qkv"]
    S, n, heads, D = x.shape
    Hkv = (heads - Hq) // 2
    k, v = c["k"].double(), c["v"].double()
    size = torch.zeros_like(k)
    q, q_size = torch.zeros(S, n, Hq, D, dtype=torch.float64), torch.zeros(S, n, Hq, D, dtype=torch.float64)
    for s in range(S):
        for i in range(n):
            place = max(int(c["lengths"][s]), 0) - n + i
            if i < first_token(c, s, n):
                continue
            new = x[s, i].double()
            mag = new.abs()
            if inv_freq is not None:
                pos = place if positions is None else int(positions[s, i])
                th = (torch.tensor(float(pos)) * inv_freq).double()          # the angle: a product of 32 bits
                cos, sin = (f(th).to(x.dtype).double().repeat(2) for f in (torch.cos, torch.sin))
                a, b = new[:Hq + Hkv, :D // 2], new[:Hq + Hkv, D // 2:]
                turned = new[:Hq + Hkv] * cos + torch.cat((-b, a), -1) * sin
                mag = mag.clone()
                mag[:Hq + Hkv] = new[:Hq + Hkv].abs() * cos.abs() + torch.cat((b, a), -1).abs() * sin.abs()
                new = torch.cat((turned, new[Hq + Hkv:]))
            q[s, i], q_size[s, i] = new[:Hq], mag[:Hq]
            at = page_of(c, s, place)
            if at is not None:
                k[at], v[at], size[at] = new[Hq:Hq + Hkv], new[Hq + Hkv:], mag[Hq:Hq + Hkv]
    return (q, q_size), (k, size), v


def attend(c, scale=None):
    """-> out, lse in float64; mean |v| under the softmax (the scale of out's sum); bound on |q| . |k| of each row's scores."""
    q = c["q"].double()
    S, n, Hq, D = q.shape
    Hkv = c["k"].shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, lse = torch.zeros(S, n, Hq, D, dtype=torch.float64), torch.full((S, Hq, n), -math.inf, dtype=torch.float64)
    mean, dots = torch.zeros_like(out), torch.zeros(S, Hq, n, dtype=torch.float64)
    for s in range(S):
        length = max(int(c["lengths"][s]), 0)
        j = torch.arange(min(length, c["table"].shape[1] * c["page"]))
        pages = c["table"][s, j // c["page"]].long()
        with_page = (pages >= 0) & (pages < c["k"].shape[0])
        j, pages = j[with_page], pages[with_page]
        if not len(j):
            continue
        K, V = c["k"][pages, j % c["page"]].double(), c["v"][pages, j % c["page"]].double()        # (keys, Hkv, D)
        for i in range(n):
            seen = j <= length - n + i
            if not seen.any() or i < first_token(c, s, n):
                continue
            for h in range(Hq):
                kk, vv = K[seen, h * Hkv // Hq], V[seen, h * Hkv // Hq]
                x = kk @ q[s, i, h] * scale
                p = torch.softmax(x, 0)
                out[s, i, h], mean[s, i, h], lse[s, h, i] = p @ vv, p @ vv.abs(), torch.logsumexp(x, 0)
                dots[s, h, i] = (kk.abs() @ q[s, i, h].abs()).max() * abs(scale)
    return out, lse, mean, dots


def attend_bounds(c, out, lse, mean, dots):
    """Largest errors that the arithmetic allows: products of the inputs are exact in 32 bits, their sum over D and the sums over the keys round
    at every addition (half a step is 2^-24), p is rounded to the values' type (half a step: eps / 2) in front of its product, the result once
    more; exp2 and the reference it is taken from are good to 2^-20 of a score of at most 100."""
    D, keys = c["q"].shape[3], max(int(c["lengths"].max()), 1)
    half = torch.finfo(c["q"].dtype).eps / 2
    x = dots * (D + 8) * 2 ** -24 + 2 ** -20
    p = 2 * x + (2 * keys + 64) * 2 ** -24 + half
    return half * out.abs() + p.transpose(1, 2)[..., None] * mean * 1.01 + 1e-30, x + (keys + 64) * 2 ** -24 + 2 ** -22 * lse.abs().nan_to_num(posinf=0) + half * 0
