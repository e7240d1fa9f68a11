"""A key / value cache in pages that holds its values in 8 bits, in 64 bits on the CPU: what tests compare the kernels with."""
import torch

import paged_reference as ref

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def to_e4m3(x):
    """float64 -> the nearest value of the type, half way to the even one; above 448, and what is not finite, NaN."""
    step = torch.exp2((torch.frexp(x)[1].double() - 1).clamp(min=-6.0) - 3.0)
    y = torch.round(x / step) * step
    return torch.where(y.abs() <= 448, y, torch.full_like(y, float("nan")))


def exponent(top):
    """The least e from -126 on with top <= 448 * 2^e."""
    e = -126
    while top > 448.0 * 2.0 ** e:
        e += 1
    return e


def byte(e):
    return torch.tensor(e + 127, dtype=torch.uint8)


def make(lengths, n, Hq, Hkv, D, page, block, dtype, seed, layout="rows"):
    """paged_reference.make with pages in 8 bits: k8, v8 of type F8, kz, vz of type E8; k, v: their values in float64, of which attention is the reference's.  What no
    token owns holds NaN, blocks without a token scales that are NaN too."""
    c = ref.make(lengths, n, Hq, Hkv, D, page, torch.float32, seed, layout=layout)
    g = torch.Generator().manual_seed(seed + 1)
    c["q"], c["qkv"], c["block"] = c["q"].to(dtype), c["qkv"].to(dtype), block
    pages = c["k"].shape[0]
    owned = torch.zeros((pages, page), dtype=torch.bool)
    for s, length in enumerate(lengths):
        for place in range(max(length, 0)):
            at = ref.page_of(c, s, place)
            if at is not None:
                owned[at] = True
    for name in ("k", "v"):
        x = c[name].double() * torch.exp(torch.randn((pages, page // block, 1, Hkv, 1), generator=g).double()).expand(-1, -1, block, -1, -1).reshape(pages, page, Hkv, 1)
        x = x * owned[:, :, None, None]
        top = x.view(pages, page // block, block, Hkv, D).abs().amax((2, 4))
        m, e = torch.frexp(top)
        e = torch.where(top > 0, e - 8 - (m <= 0.875).int(), torch.full_like(e, -126))
        assert all(exponent(float(t)) == int(k) for t, k in zip(top.flatten()[:50], e.flatten()[:50]))
        scale = torch.exp2(e.double()).repeat_interleave(block, 1)[..., None]
        held = to_e4m3(x / scale)
        c[name] = held * scale
        held[~owned] = float("nan")
        bytes_ = (e + 127).to(torch.uint8)
        bytes_[~owned.view(pages, page // block, block).any(2)] = 255
        # the storage's layout: that of the values for the pages, heads outside of blocks for a layout with heads outside of rows
        like = torch.empty_strided(c[name].shape, _strides(c[name].shape, layout), dtype=F8)
        like.view(torch.uint8).copy_(held.float().to(F8).view(torch.uint8))
        c[name + "8"] = like
        z = torch.empty((pages, Hkv, page // block), dtype=E8).transpose(1, 2) if layout == "heads" else torch.empty((pages, page // block, Hkv), dtype=E8)
        z.view(torch.uint8).copy_(bytes_)
        c[name + "z"] = z
    return c


def _strides(shape, layout):
    pages, page, Hkv, D = shape
    if layout == "heads":
        return (Hkv * page * D, D, page * D, 1)
    if layout == "mixed":      # a wider row of heads, and something between pages
        return (page * (Hkv + 1) * D + 48, (Hkv + 1) * D, D, 1)
    return (page * Hkv * D, Hkv * D, D, 1)


def cache(g):
    return g["k8"], g["v8"], g["kz"], g["vz"], g["table"], g["lengths"]


def append(c, Hq, inv_freq=None, positions=None):
    """-> q as paged_reference.append has it; for keys and values what is to be stored: (bytes of the pages, bytes of the scales, unrounded values in float64 where a
    new token has them else NaN, sizes of the products in them)."""
    wide = dict(c, k=torch.full(c["k8"].shape, float("nan"), dtype=torch.float64), v=torch.full(c["v8"].shape, float("nan"), dtype=torch.float64))
    (q, q_size), (k, size), v = ref.append(wide, Hq, inv_freq, positions)
    n, b = c["qkv"].shape[1], c["block"]
    out = []
    for new, old, z in ((k, c["k8"], c["kz"]), (v, c["v8"], c["vz"])):
        rows, scales = old.clone().view(torch.uint8), z.clone().view(torch.uint8)
        rounded = new.float().double()
        for s in range(c["qkv"].shape[0]):
            length = max(int(c["lengths"][s]), 0)
            first = length - n + ref.first_token(c, s, n)
            for j in range(first // b, (length + b - 1) // b) if first < length else ():
                at = ref.page_of(c, s, j * b)
                if at is None:
                    continue
                page, r0 = at
                since, end = max(first, j * b) - j * b + r0, min(length, j * b + b) - j * b + r0
                for h in range(old.shape[2]):
                    x = rounded[page, since:end, h]
                    top = x[torch.isfinite(x)].abs().max() if torch.isfinite(x).any() else torch.zeros(())
                    e = exponent(float(top))
                    if since > r0:
                        before = int(scales[page, r0 // b, h]) - 127
                        e = max(e, before)
                        moved = to_e4m3(old[page, r0:since, h].double() * 2.0 ** (before - e))
                        rows[page, r0:since, h] = moved.float().to(F8).view(torch.uint8)
                    rows[page, since:end, h] = to_e4m3(x * 2.0 ** -e).float().to(F8).view(torch.uint8)
                    scales[page, r0 // b, h] = e + 127
        out.append((rows, scales, new))
    return (q, q_size), (*out[0], size), out[1]


def values(rows, scales, block):
    """float64 values of pages and scales."""
    return rows.view(F8).double() * torch.exp2(scales.view(torch.uint8).double() - 127).repeat_interleave(block, 1)[..., None]
