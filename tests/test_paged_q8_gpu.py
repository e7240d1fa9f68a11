"""A key / value cache in pages that holds its values in 8 bits: appending, reading back, attention over it, against 64 bits on the CPU."""
import math

import pytest
import torch

import paged_q8_reference as q8
import paged_reference as ref
from paged_q8_reference import E8, F8

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _to(c, dev):
    def move(t):   # keeps the strides: what is tested with a layout is that layout
        to = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev)
        if t.dtype in (F8, E8):
            to.view(torch.uint8).copy_(t.view(torch.uint8))
            return to
        return to.copy_(t)
    return {k: move(t) if torch.is_tensor(t) and k not in ("k", "v") else t for k, t in c.items()}


def _inv_freq(D, base=10000.0):
    return 1.0 / (base ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D))


def _bytes(t):
    return t.view(torch.uint8).cpu()


def _rows(t):
    """Bytes of pages; a NaN has either sign."""
    b = t.view(torch.uint8).cpu()
    return torch.where(b & 0x7f == 0x7f, 0x7f, b)


def _check_append(c, dev, Hq, positions=None, rotate=True):
    from odysseus_transformer_amd import ops
    g = _to(c, dev)
    dtype, D, b = c["q"].dtype, c["q"].shape[3], c["block"]
    f = _inv_freq(D)
    (q, q_size), (k_rows, k_scales, k_new, size), (v_rows, v_scales, v_new) = q8.append(c, Hq, f if rotate else None, positions)
    k_rows, v_rows = _rows(k_rows), _rows(v_rows)
    qkv = g["qkv"].clone()
    got = ops.paged_append_q8_(g["qkv"], Hq, *q8.cache(g), position_ids=None if positions is None else positions.to(dev),
                               inv_freq=f.to(dev) if rotate else None, rotate=rotate, new_tokens=g.get("new"))
    torch.cuda.synchronize()
    bits = torch.int16 if dtype == BF16 else torch.int32   # NaN is not equal to itself
    assert torch.equal(g["qkv"].view(bits), qkv.view(bits)), "the projection was written to"
    assert torch.equal(_bytes(g["vz"]), v_scales), "scales of values"
    assert torch.equal(_rows(g["v8"]), v_rows), "values"
    if not rotate:
        assert got.data_ptr() == g["qkv"].data_ptr() and torch.equal(got.view(bits), qkv[:, :, :Hq].view(bits))
        assert torch.equal(_bytes(g["kz"]), k_scales), "scales of keys"
        assert torch.equal(_rows(g["k8"]), k_rows), "keys"
        return g
    half = torch.finfo(dtype).eps / 2
    have = got.double().cpu()
    assert torch.equal(have[q_size == 0], q[q_size == 0])
    # one rounding, the sum's in 32 bits, and a cosine next to the middle of two values of the type, which may round to either one
    assert ((have - q).abs() <= half * q.abs() + (2 * half + 2 ** -22) * q_size).all(), "q"
    # keys: the same in front of the eight bits, of which a half step is 2^-4 of a value, or 2^-10 of the scale below 2^-6 of it.  The scale is that of the largest value, which may be
    # off as much: where it is next to a border either exponent
    kz, k8 = _bytes(g["kz"]), _rows(g["k8"])
    off = kz.int() - k_scales.int()
    assert (off.abs() <= 1).all() and (off != 0).double().mean() < 0.01, "scales of keys"
    scale = torch.exp2(torch.maximum(kz, k_scales).double() - 127).repeat_interleave(b, 1)[..., None]
    held, new = q8.values(k8, kz, b), torch.isfinite(k_new)
    err = (held - k_new).abs()
    slack = (2 * half + 2 ** -22) * size
    assert (err <= torch.maximum(2 ** -4 * (k_new.abs() + slack), 2 ** -10 * scale) + slack)[new].all(), "keys"
    assert (k8 != k_rows)[new].sum() <= 0.01 * new.sum(), "keys are not the nearest values"
    same = (off == 0).repeat_interleave(b, 1)[..., None].expand_as(new) & ~new
    assert torch.equal(k8[same], k_rows[same]), "rows without a new token"
    return g


APPEND = [
    # lengths, n, Hq, Hkv, D, page, block, dtype, layout
    ([1], 1, 1, 1, 128, 16, 16, BF16, "rows"),
    ([5, 0, 17, 33, 8], 1, 4, 2, 128, 8, 8, BF16, "rows"),            # a sequence that takes no part
    ([9, 3, 40], 9, 8, 2, 64, 16, 8, BF16, "heads"),                  # padded on the left
    ([300, 131, 70], 67, 6, 3, 128, 32, 16, BF16, "mixed"),
    ([100, 20], 33, 5, 1, 64, 64, 64, F32, "rows"),
    ([41, 0, 1], 7, 4, 4, 128, 8, 8, F32, "mixed"),
    ([2, 1], 2, 8, 8, 64, 256, 32, F32, "heads"),
    ([700], 700, 4, 1, 128, 128, 64, BF16, "rows"),
    ([90, 63, 64, 65, 1], 1, 5, 5, 64, 64, 32, BF16, "heads"),
    ([90, 63, 64, 65, 1], 1, 3, 3, 128, 64, 64, F32, "heads"),
    ([150, 31], 64, 2, 2, 128, 64, 64, F32, "rows"),
    (list(range(1, 98)), 1, 2, 1, 64, 16, 16, BF16, "rows"),
    ([33, 12], 3, 40, 40, 64, 32, 32, BF16, "rows"),
]
_ids = lambda c: "S%d_max%d_n%d_H%d_%d_D%d_p%d_b%d_%s_%s" % (len(c[0]), max(c[0]), *c[1:7], str(c[7])[-4:], c[8])  # noqa: E731


@pytest.mark.parametrize("case", APPEND, ids=_ids)
def test_append(case, dev):
    lengths, n, Hq, Hkv, D, page, block, dtype, layout = case
    print(f"append {case}", flush=True)
    c = q8.make(lengths, n, Hq, Hkv, D, page, block, dtype, seed=n + Hq, layout=layout)
    _check_append(c, dev, Hq)
    _check_append(c, dev, Hq, rotate=False)


@pytest.mark.parametrize("n", [1, 2, 5])
@pytest.mark.parametrize("dtype,D,block", [(BF16, 128, 32), (BF16, 64, 64), (F32, 128, 16), (F32, 64, 8)], ids=lambda x: str(x)[-4:])
def test_scales_rise_with_larger_tokens(n, dtype, D, block, dev):
    """New tokens far above, and far below, the earlier ones of their block: those are rounded to the new scale, down to nothing, or keep it."""
    c = q8.make([block + 5, 3, 2 * block - 1, block + 1, block, 40], n, 4, 2, D, 64, block, dtype, seed=n + D)
    size = torch.tensor([2.0 ** 4, 2.0 ** -5, 2.0 ** 9, 2.0 ** 14, 2.0 ** 30, 2.0 ** -140]).view(-1, 1, 1, 1)
    c["qkv"] = (c["qkv"].float() * size).to(dtype)
    _check_append(c, dev, 4, rotate=False)


def test_borders_of_scales_and_values(dev):
    """A largest value on a border of two scales and next to it; halfway cases of the eight bits; values of the smallest sizes; zeros."""
    c = q8.make([16, 16, 16, 16, 16, 16], 16, 1, 1, 64, 16, 16, F32, seed=1)
    x = torch.zeros((6, 16, 3, 64))
    grid = torch.arange(0, 448.25, 0.25)
    x[0].view(-1)[:grid.numel()] = grid                                              # every value, and every middle of two
    x[1, :, :, 0], x[1, 0, :, 1] = 448.0, -448.0
    x[2, 0, :, 0] = math.nextafter(448.0, 512.0) + 2 ** -15
    x[3] = torch.randn((16, 3, 64), generator=torch.Generator().manual_seed(5)) * 2.0 ** -128   # below the smallest normal numbers
    x[4, 0, :, 0], x[4, 1, :, :] = 2.0 ** 127 * 1.75, -(2.0 ** 127)
    c["qkv"] = x
    g = _check_append(c, dev, 1, rotate=False)
    assert (g["vz"].view(torch.uint8)[c["table"][5, 0].item()] == 1).all()          # nothing but zeros: the smallest scale


def test_infinite_and_nan_values(dev):
    """They become NaN, and the scale is that of the others."""
    for n, lengths in ((1, [20, 1]), (24, [24, 30])):
        c = q8.make(lengths, n, 2, 2, 64, 16, 16, BF16, seed=n)
        c["qkv"][0, -1, 3, 5], c["qkv"][0, -1, 5, 60], c["qkv"][1, -1, 4, 0] = math.inf, -math.inf, math.nan
        g = _check_append(c, dev, 2, rotate=False)
        held = q8.values(_rows(g["v8"]), _bytes(g["vz"]), 16)
        p, r = ref.page_of(c, 1, lengths[1] - 1)
        assert torch.isnan(held[p, r, 0, 0]) and torch.isfinite(held[p, r, 0, 1:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_append_with_positions_of_its_own(dtype, dev):
    c = q8.make([50, 11, 30], 4, 4, 2, 128, 16, 8, dtype, seed=3)
    own = torch.tensor([[131071, 0, 7, 99999], [1, 2, 3, 4], [65536, 65537, 12, 0]])
    _check_append(c, dev, 4, positions=own)
    from odysseus_transformer_amd import ops
    g, h = _to(c, dev), _to(c, dev)
    shared = torch.tensor([3, 4, 5, 6], device=dev)
    a = ops.paged_append_q8_(g["qkv"], 4, *q8.cache(g), position_ids=shared)
    b = ops.paged_append_q8_(h["qkv"], 4, *q8.cache(h), position_ids=shared.to(torch.int32).expand(3, 4).contiguous())
    assert torch.equal(a, b) and torch.equal(_rows(g["k8"]), _bytes(h["k8"]))


def test_queries_are_those_of_the_other_cache(dev):
    """But for cosines that are rounded from 64 bits here and from 32 there: a step of the type of one of them, in either product, and the result's rounding."""
    from odysseus_transformer_amd import ops
    for dtype in (BF16, F32):
        c = q8.make([77, 77, 5], 77, 6, 2, 128, 16, 16, dtype, seed=8)
        g = _to(c, dev)
        k, v = (torch.zeros(c["k8"].shape, dtype=dtype, device=dev) for _ in range(2))
        a = ops.paged_append_(g["qkv"], 6, k, v, g["table"], g["lengths"]).double()
        b = ops.paged_append_q8_(g["qkv"], 6, *q8.cache(g)).double()
        x = g["qkv"][:, :, :6].double().abs()
        size = x + torch.cat((x[..., 64:], x[..., :64]), -1)
        eps = torch.finfo(dtype).eps
        assert ((a - b).abs() <= eps * size + eps * a.abs()).all()
        assert (a == b).double().mean() > (0.99 if dtype == BF16 else 0.5)


@pytest.mark.parametrize("dtype,n", [(BF16, 2801), (F32, 1403)], ids=["bf16", "f32"])
def test_large_projections_are_appended_as_small_ones(dtype, n, dev):
    """A projection of more than 128 MB is read in another way: the same bytes as sequence by sequence."""
    from odysseus_transformer_amd import ops
    S, Hq, Hkv, D, page, block = 4, 32, 8, 128, 64, 32
    assert S * n * (Hq + 2 * Hkv) * D * (2 if dtype == BF16 else 4) >= 128e6
    lengths = torch.tensor([n, n + 45, 700, n + 7], dtype=torch.int32, device=dev)
    columns = (n + 45 + page - 1) // page
    table = torch.randperm(S * columns, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(S, columns).to(dev)
    qkv = torch.randn((S, n, Hq + 2 * Hkv, D), generator=torch.Generator(device=dev).manual_seed(2), device=dev).to(dtype)

    def caches():
        return tuple(torch.zeros((S * columns, page, Hkv, D), dtype=torch.uint8, device=dev).view(F8) for _ in range(2)) + \
            tuple(torch.full((S * columns, page // block, Hkv), 120, dtype=torch.uint8, device=dev).view(E8) for _ in range(2))
    for rotate in (True, False):
        a, b = caches(), caches()
        q = ops.paged_append_q8_(qkv, Hq, *a, table, lengths, rotate=rotate)
        for s in range(S):
            one = ops.paged_append_q8_(qkv[s:s + 1], Hq, *b, table[s:s + 1], lengths[s:s + 1], rotate=rotate)
            assert torch.equal(one[0], q[s])
        for x, y in zip(a, b):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_cosines_are_rounded_to_32_bits_first(dev):
    """Queries of 1 and 0 are the cosines and sines: those of 32 bits, rounded once more to the type.  (Among 2^19 of them a few lie in the middle of two bf16 values then.)"""
    from odysseus_transformer_amd import ops
    n, D = 4096, 128
    c = q8.make([n], n, 1, 1, D, 64, 32, BF16, seed=1)
    g = _to(c, dev)
    g["qkv"][:, :, 0, :D // 2], g["qkv"][:, :, 0, D // 2:] = 1.0, 0.0
    q = ops.paged_append_q8_(g["qkv"], 1, *q8.cache(g), inv_freq=_inv_freq(D).to(dev))[0, :, 0].cpu()
    th = (torch.arange(n).float()[:, None] * _inv_freq(D)).double()
    assert torch.equal(q, torch.cat((th.cos(), th.sin()), -1).float().to(BF16))


NEW = [
    # lengths, new tokens, n, Hq, Hkv, D, page, block, dtype
    ([40, 300, 7, 90], [1, 1, 0, 1], 1, 8, 2, 128, 16, 8, BF16),
    ([40, 300, 7, 90, 3], [5, 0, 2, 9, -1], 5, 4, 2, 64, 8, 8, BF16),               # more than n, fewer than none
    ([150, 300, 100, 20], [64, 1, 0, 20], 64, 4, 1, 128, 32, 32, BF16),              # tiles of a sequence without a token in front
    ([270, 90, 200], [1, 80, 66], 80, 2, 1, 64, 64, 64, BF16),
    ([40, 300, 7, 90], [1, 0, 1, 0], 1, 4, 2, 64, 16, 16, F32),
    ([90, 200, 33], [33, 2, 0], 33, 4, 1, 128, 8, 8, F32),
    ([500, 60], [0, 0], 100, 4, 2, 128, 16, 16, BF16),                               # nobody
]


@pytest.mark.parametrize("case", NEW, ids=lambda c: "n%d_H%d_%d_D%d_p%d_b%d_%s" % (*c[2:8], str(c[8])[-4:]))
def test_sequences_with_fewer_new_tokens(case, dev):
    lengths, new, n, Hq, Hkv, D, page, block, dtype = case
    print(f"new {case}", flush=True)
    c = q8.make(lengths, n, Hq, Hkv, D, page, block, dtype, seed=n + D)
    c["new"] = torch.tensor(new, dtype=torch.int32)
    _check_attn(c, _to(c, dev))
    _check_append(c, dev, Hq)
    _check_append(c, dev, Hq, rotate=False)


# ------------------------------------------------------------------------------------------------ reading back
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lengths,Hkv,D,page,block,layout", [([1], 1, 64, 8, 8, "rows"), ([70, 0, 33, -2], 3, 128, 32, 16, "heads"), ([900, 17], 5, 64, 64, 64, "mixed"),
                                                             ([40] * 70, 2, 128, 16, 8, "heads")])
def test_read(lengths, Hkv, D, page, block, layout, dtype, dev):
    from odysseus_transformer_amd import ops
    c = q8.make(lengths, 1, Hkv, Hkv, D, page, block, dtype, seed=D + Hkv, layout=layout)
    if len(lengths) > 1:
        c["table"][0, 1] = -1
        c["table"][-1, 0] = c["k8"].shape[0]
    g = _to(c, dev)
    for places in sorted({1, max(lengths), max(lengths) + 3, c["table"].shape[1] * page + 5}):
        k, v = ops.paged_read_q8(*q8.cache(g), places, dtype)
        for have, want in ((k, c["k"]), (v, c["v"])):
            expect = torch.zeros((len(lengths), places, Hkv, D), dtype=torch.float64)
            for s, length in enumerate(lengths):
                for place in range(min(max(length, 0), places)):
                    at = ref.page_of(c, s, place)
                    if at is not None:
                        expect[s, place] = want[at]
            assert have.dtype == dtype and torch.equal(have.double().cpu(), expect)
    k, v = ops.paged_read_q8(*q8.cache(g), 0, dtype)
    assert k.shape == v.shape == (len(lengths), 0, Hkv, D)


# ------------------------------------------------------------------------------------------------ attention
def _check_attn(c, g, scale=None):
    from odysseus_transformer_amd import ops
    out, lse = ops.paged_attn_q8(g["q"], *q8.cache(g), scale=scale, new_tokens=g.get("new"))
    torch.cuda.synchronize()
    o, s, mean, dots = ref.attend(c, scale)
    tol_o, tol_s = ref.attend_bounds(c, o, s, mean, dots)
    out, lse = out.double().cpu(), lse.double().cpu()
    none = s == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert (out[none.transpose(1, 2)] == 0).all()
    bad = ~((out - o).abs() <= tol_o)
    assert not bad.any(), f"out: {int(bad.sum())} of {bad.numel()} beyond their bounds, worst {((out - o).abs() / tol_o).max():.2f}"
    bad = ~((lse - s).abs() <= tol_s) & ~none
    assert not bad.any(), f"lse: {int(bad.sum())} beyond their bounds, worst {((lse - s).abs()[~none] / tol_s[~none]).max():.2f}"


ATTN = [
    # lengths, n, Hq, Hkv, D, page, block, dtype, layout
    ([1], 1, 1, 1, 128, 16, 16, BF16, "rows"),
    ([1], 1, 1, 1, 64, 8, 8, F32, "rows"),
    ([100], 1, 4, 1, 128, 16, 8, BF16, "rows"),
    ([5, 0, 17, 33, 8, 128, 129, 127, 31, 32, 255, 256, 257], 1, 4, 2, 128, 8, 8, BF16, "rows"),
    ([700, 1, 64, 1029], 1, 8, 2, 64, 32, 16, BF16, "heads"),
    ([2000, 513, 4], 1, 32, 8, 128, 64, 32, BF16, "mixed"),
    ([600, 77], 1, 32, 1, 128, 16, 16, BF16, "rows"),                 # 32 rows of one kv head
    ([600, 77], 1, 40, 1, 64, 16, 16, BF16, "rows"),                  # 40
    ([400, 70], 1, 71, 1, 128, 64, 64, BF16, "rows"),                 # 71
    ([300, 2], 5, 7, 1, 128, 16, 8, BF16, "rows"),                    # 35 rows, padded on the left
    ([150, 40, 3, 0], 8, 8, 8, 64, 16, 16, BF16, "heads"),
    ([333], 333, 4, 1, 128, 32, 32, BF16, "rows"),                    # a whole prompt
    ([400, 90, 200], 130, 6, 2, 128, 64, 16, BF16, "mixed"),
    ([260, 129], 65, 4, 4, 64, 8, 8, BF16, "rows"),
    ([500, 33, 1, 0], 1, 8, 8, 64, 32, 32, F32, "rows"),
    ([290, 40], 1, 24, 2, 128, 16, 8, F32, "heads"),
    ([129, 64, 31], 6, 6, 2, 64, 8, 8, F32, "mixed"),
    ([150, 20], 40, 4, 2, 128, 64, 64, F32, "rows"),
    ([4096 + 3], 1, 8, 8, 128, 128, 64, BF16, "rows"),
    ([3000], 1, 2, 2, 64, 256, 64, F32, "rows"),
    (list(range(0, 260, 2)), 1, 2, 1, 64, 16, 16, BF16, "rows"),      # more sequences than a wavefront has lanes
]


@pytest.mark.parametrize("D,page,block", [(128, 64, 32), (64, 16, 16), (128, 8, 8), (64, 64, 64)])
def test_tiles_of_256_rows(D, page, block, dev):
    """Row tiles of 256, of 64 (sequence, kv head) pairs: lengths around tiles of keys, short and padded sequences, pages of one group of keys and of a tile; all
    rows of some of the sequences."""
    from odysseus_transformer_amd import ops
    lengths, n, Hq, Hkv = [200, 128, 321, 130, 64, 191, 1, 0], 128, 16, 8
    c = q8.make(lengths, n, Hq, Hkv, D, page, block, BF16, seed=D + page)
    c["table"][2, 1] = -1
    g = _to(c, dev)
    out, lse = ops.paged_attn_q8(g["q"], *q8.cache(g))
    for heads in (slice(0, 2), slice(14, 16)):
        part = dict(c, q=c["q"][:, :, heads], k=c["k"][:, :, heads.start // 2:heads.start // 2 + 1], v=c["v"][:, :, heads.start // 2:heads.start // 2 + 1])
        o, s, mean, dots = ref.attend(part)
        tol_o, tol_s = ref.attend_bounds(part, o, s, mean, dots)
        none = s == -math.inf
        assert ((out[:, :, heads].double().cpu() - o).abs() <= tol_o).all()
        assert torch.equal(lse[:, heads].cpu() == -math.inf, none) and ((lse[:, heads].double().cpu() - s).abs() <= tol_s)[~none].all()


def _check_heads(c, g, dev, heads, **kw):
    """Some query heads of a case with one for each kv head."""
    from odysseus_transformer_amd import ops
    out, lse = ops.paged_attn_q8(g["q"], *q8.cache(g), **kw)
    for h in heads:
        part = dict(c, q=c["q"][:, :, h:h + 1], k=c["k"][:, :, h:h + 1], v=c["v"][:, :, h:h + 1])
        o, s, mean, dots = ref.attend(part)
        tol_o, tol_s = ref.attend_bounds(part, o, s, mean, dots)
        none = s == -math.inf
        assert ((out[:, :, h:h + 1].double().cpu() - o).abs() <= tol_o).all(), h
        assert torch.equal(lse[:, h:h + 1].cpu() == -math.inf, none) and ((lse[:, h:h + 1].double().cpu() - s).abs() <= tol_s)[~none].all(), h


@pytest.mark.parametrize("n,D", [(256, 128), (128, 128), (128, 64)], ids=["256", "128", "128_hd64"])
@pytest.mark.parametrize("length", [1, 8, 64, 65, 71, 128, 129, 192, 193, 256, 257, 320, 321, 520, 1100])
def test_many_rows_of_few_tiles(length, n, D, dev):
    """As many tiles of keys as a loop over them can begin and end with, and groups of keys with one, all or none of theirs there; a page that is not there."""
    c = q8.make([length], n, 64, 64, D, 16, 8, BF16, seed=length)
    if length > 100:
        c["table"][0, 5] = -1
    _check_heads(c, _to(c, dev), dev, (0, 37, 63))


@pytest.mark.parametrize("n", [256, 128])
def test_many_rows_with_fewer_new_tokens(n, dev):
    c = q8.make([300, 40, 500], n, 64, 64, 128, 16, 16, BF16, seed=n)
    c["new"] = torch.tensor([90, 0, n - 1], dtype=torch.int32)
    g = _to(c, dev)
    _check_heads(c, g, dev, (2, 63), new_tokens=g["new"])


@pytest.mark.parametrize("n", [256, 128])
def test_many_rows_whose_scores_grow(n, dev):
    c = q8.make([1000], n, 64, 64, 128, 32, 8, BF16, seed=3)
    up = torch.arange(c["table"].shape[1]) // 3
    z = c["kz"].view(torch.uint8)
    for col in range(c["table"].shape[1]):
        pg = int(c["table"][0, col])
        z[pg] = torch.where(z[pg] == 255, 255, z[pg].int() + int(up[col])).to(torch.uint8)
    held = c["k8"].double()
    c["k"] = torch.where(torch.isnan(held), 0.0, held) * torch.where(z == 255, 1.0, torch.exp2(z.double() - 127)).repeat_interleave(8, 1)[..., None]
    _check_heads(c, _to(c, dev), dev, (0, 1, 40))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[64], [65, 1], [128, 63], [192, 191], [321, 448, 64], [130 + 64 * 9]], ids=str)
def test_chunks_of_few_tiles(D, lengths, dev):
    """As many tiles of keys as a loop with several of them in flight can begin and end with."""
    for n in (65, 200):
        c = q8.make(lengths, n, 2, 1, D, 8, 8, BF16, seed=sum(lengths) + n)
        _check_attn(c, _to(c, dev))


@pytest.mark.parametrize("n", [1, 66], ids=["one", "chunk"])
def test_scores_that_grow(n, dev):
    """Later keys far above the earlier ones: references follow."""
    c = q8.make([900, 300], n, 4, 2, 128, 16, 8, BF16, seed=n)
    grow = torch.exp2(torch.arange(0, 57 + n // 66 * 4) // 8)[: (900 + 15) // 16]
    for s in range(2):
        for col in range(c["table"].shape[1]):
            pg = int(c["table"][s, col])
            if pg >= 0:
                z = c["kz"].view(torch.uint8)[pg].int() + int(torch.log2(grow[min(col, len(grow) - 1)]))
                live = c["kz"].view(torch.uint8)[pg] != 255
                c["kz"].view(torch.uint8)[pg] = torch.where(live, z.to(torch.uint8), 255)
    c["k"] = torch.where(torch.isnan(c["k8"].double()), 0.0, c["k8"].double()) * torch.where(
        c["kz"].view(torch.uint8) == 255, 1.0, torch.exp2(c["kz"].view(torch.uint8).double() - 127)).repeat_interleave(8, 1)[..., None]
    _check_attn(c, _to(c, dev))


@pytest.mark.parametrize("case", ATTN, ids=_ids)
def test_attn(case, dev):
    lengths, n, Hq, Hkv, D, page, block, dtype, layout = case
    print(f"attn {case}", flush=True)
    c = q8.make(lengths, n, Hq, Hkv, D, page, block, dtype, seed=n + Hq + D, layout=layout)
    _check_attn(c, _to(c, dev))


@pytest.mark.parametrize("many_rows", [False, True], ids=["few_rows", "many_rows"])
def test_scale_and_strided_queries(many_rows, dev):
    n = 70 if many_rows else 3
    c = q8.make([90, 200], n, 4, 2, 128, 16, 8, BF16, seed=1)
    g = _to(c, dev)
    for scale in (0.25, 0.0, -0.1):
        _check_attn(c, g, scale)
    c["q"] = c["qkv"][:, :, :4]
    g["q"] = g["qkv"][:, :, :4]                                   # a slice of the packed projection
    _check_attn(c, g)


@pytest.mark.parametrize("n,Hq,Hkv,D,dtype", [(1, 8, 2, 128, BF16), (9, 4, 1, 64, BF16), (70, 4, 2, 128, BF16), (300, 2, 1, 128, BF16), (130, 2, 1, 64, BF16), (1, 4, 4, 128, F32)],
                         ids=lambda x: str(x)[-4:])
def test_entries_that_are_no_page(n, Hq, Hkv, D, dtype, dev):
    """Their keys take no part, nothing is read or written there."""
    c = q8.make([n + 60, n + 150, n + 3], n, Hq, Hkv, D, 8, 8, dtype, seed=n)
    for s, column, entry in ((0, 0, -1), (0, 4, 1 << 30), (1, 7, -5), (1, (n + 149) // 8, c["k8"].shape[0]), (2, 0, -1 << 31)):
        c["table"][s, column] = entry
    _check_attn(c, _to(c, dev))
    _check_append(c, dev, Hq, rotate=False)


def test_sequences_that_share_pages(dev):
    c = q8.make([300, 290, 300], 1, 4, 2, 128, 16, 16, BF16, seed=4)
    c["table"][1, :16] = c["table"][0, :16]
    c["table"][2] = c["table"][0]
    _check_attn(c, _to(c, dev))


@pytest.mark.parametrize("n", [1, 80])
def test_nan_values_reach_their_own_head_only(n, dev):
    from odysseus_transformer_amd import ops
    c = q8.make([200, 150], n, 4, 2, 128, 16, 16, BF16, seed=n)
    g = _to(c, dev)
    clean, clean_lse = ops.paged_attn_q8(g["q"], *q8.cache(g))
    p, r = ref.page_of(c, 0, 20)
    g["v8"][p, r, 0, 3:4].view(torch.uint8).fill_(0x7f)
    out, lse = ops.paged_attn_q8(g["q"], *q8.cache(g))
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, :, :2, 3] = True
    assert torch.equal(torch.isnan(out), hit) and torch.equal(out[~hit], clean[~hit]) and torch.equal(lse, clean_lse)


def test_attends_what_was_appended_step_by_step(dev):
    """A prompt, then single tokens and a few at once, into one cache: every step against 64 bits over what the cache holds."""
    from odysseus_transformer_amd import ops
    Hq, Hkv, D, page, block, dtype = 8, 2, 128, 32, 16, BF16
    c = q8.make([120, 90], 1, Hq, Hkv, D, page, block, dtype, seed=2)
    g = _to(c, dev)
    gen = torch.Generator().manual_seed(9)
    lengths = torch.zeros(2, dtype=torch.int32)
    for new in ([70, 41], [1, 1], [1, 0], [5, 5], [1, 1], [3, 7], [1, 1]):
        n = max(new)
        lengths += torch.tensor(new, dtype=torch.int32)
        c["lengths"], c["new"] = lengths.clone(), torch.tensor(new, dtype=torch.int32)
        c["qkv"] = torch.randn((2, n, Hq + 2 * Hkv, D), generator=gen).to(dtype) * 2.0 ** (len(new) - n % 5)
        g.update({k: c[k].to(dev) for k in ("lengths", "new", "qkv")})
        q = ops.paged_append_q8_(g["qkv"], Hq, *q8.cache(g), new_tokens=g["new"])
        g["q"], c["q"] = q, q.cpu()
        for name in ("k", "v"):
            c[name] = q8.values(_bytes(g[name + "8"]), _bytes(g[name + "z"]), block)
        _check_attn(c, g)


def test_both_host_paths_agree(dev, monkeypatch):
    from odysseus_transformer_amd import _native, ops
    c = q8.make([90, 33], 3, 4, 2, 128, 32, 16, BF16, seed=6)

    def all_of():
        g = _to(c, dev)
        q = ops.paged_append_q8_(g["qkv"], 4, *q8.cache(g))
        q2 = ops.paged_append_q8_(g["qkv"], 4, *q8.cache(g), rotate=False)
        return [q, q2, *ops.paged_read_q8(*q8.cache(g), 70), *ops.paged_read_q8(*q8.cache(g), 70, F32), *ops.paged_attn_q8(q, *q8.cache(g)), g["k8"].view(torch.uint8),
                g["kz"].view(torch.uint8)]
    plain = all_of()
    monkeypatch.setattr(ops, "native", _native._Nothing())
    for a, b in zip(plain, all_of()):
        assert torch.equal(a, b)


def test_replayed_from_a_graph_with_other_lengths_and_pages(dev):
    """A captured step of append, attention and reading back replays with what the table and the lengths hold then; eager work between the replays."""
    from odysseus_transformer_amd import ops
    c = q8.make([300, 200, 40], 1, 8, 2, 128, 16, 8, BF16, seed=5)
    g, h = _to(c, dev), _to(c, dev)

    def step(x):
        q = ops.paged_append_q8_(x["qkv"], 8, *q8.cache(x))
        return (q, *ops.paged_attn_q8(q, *q8.cache(x)), *ops.paged_read_q8(*q8.cache(x), 320))
    lengths = g["lengths"].clone()
    g["lengths"].copy_(torch.tensor([1, 1, 1], dtype=torch.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    spare = _to(c, dev)
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(g)
    for turn in range(3):
        now = lengths - torch.tensor([0, 50 * turn, turn], dtype=torch.int32, device=dev)
        for x in (g, h):
            x["lengths"].copy_(now)
            x["qkv"].copy_((c["qkv"].float() * (turn + 1)).to(BF16))
            if turn == 2:
                x["table"][0].copy_(x["table"][1])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(h)):   # in the last turn sequence 0 sees rows that nobody owns, which hold NaN
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num()), turn
        assert torch.equal(_rows(g["k8"]), _bytes(h["k8"])) and torch.equal(_bytes(g["vz"]), _bytes(h["vz"]))


def test_calls_on_two_streams_at_once(dev):
    from odysseus_transformer_amd import ops
    cs = [q8.make([2000 - 300 * i, 900], 1, 8, 2, 128, 64, 32, BF16, seed=i) for i in range(2)]
    gs = [_to(c, dev) for c in cs]
    want = [ops.paged_attn_q8(g["q"], *q8.cache(g)) for g in gs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in gs]
    got = []
    for _ in range(3):
        for g, st in zip(gs, streams):
            with torch.cuda.stream(st):
                got.append(ops.paged_attn_q8(g["q"], *q8.cache(g)))
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(l, want[i % 2][1])


@pytest.mark.parametrize("n", [1, 70], ids=["one", "chunk"])
def test_offsets_beyond_32_bits(n, dev):
    """Pages more than 4 GiB behind the pool's first one."""
    from odysseus_transformer_amd import ops
    page, Hkv, D, block = 64, 8, 128, 64
    pages = (1 << 32) // (page * Hkv * D) + 40
    pool = torch.empty((2, pages, page, Hkv, D), dtype=F8, device=dev)
    c = q8.make([150, 100], n, 16, Hkv, D, page, block, BF16, seed=1)
    g = _to(c, dev)
    scales = torch.empty((2, pages, 1, Hkv), dtype=E8, device=dev)
    small = c["k8"].shape[0]
    for i, name in enumerate(("k", "v")):
        pool[i, -small:].view(torch.uint8).copy_(g[name + "8"].view(torch.uint8))
        scales[i, -small:].view(torch.uint8).copy_(g[name + "z"].view(torch.uint8))
    want = ops.paged_attn_q8(g["q"], *q8.cache(g))
    table = torch.where(g["table"] >= 0, g["table"] + (pages - small), g["table"]).to(torch.int32)
    got = ops.paged_attn_q8(g["q"], pool[0], pool[1], scales[0], scales[1], table, g["lengths"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ops.paged_append_q8_(g["qkv"], 16, *q8.cache(g))
    ops.paged_append_q8_(g["qkv"], 16, pool[0], pool[1], scales[0], scales[1], table, g["lengths"])
    assert torch.equal(pool[0, -small:].view(torch.uint8), g["k8"].view(torch.uint8)) and torch.equal(scales[1, -small:].view(torch.uint8), g["vz"].view(torch.uint8))
    for a, b in zip(ops.paged_read_q8(*q8.cache(g), 150), ops.paged_read_q8(pool[0], pool[1], scales[0], scales[1], table, g["lengths"], 150)):
        assert torch.equal(a, b)


def test_nothing_to_do(dev):
    from odysseus_transformer_amd import ops
    c = q8.make([20, 3], 1, 4, 2, 64, 16, 16, BF16, seed=1)
    g = _to(c, dev)
    before = _rows(g["k8"]).clone()
    assert ops.paged_append_q8_(g["qkv"][:, :0], 4, *q8.cache(g)).shape == (2, 0, 4, 64)
    out, lse = ops.paged_attn_q8(g["q"][:, :0], *q8.cache(g))
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    assert torch.equal(_rows(g["k8"]), before)


def test_refusals(dev):
    from odysseus_transformer_amd import _lib, ops
    c = q8.make([20, 3], 1, 4, 2, 64, 16, 8, BF16, seed=1)
    g = _to(c, dev)
    good = dict(k_pages=g["k8"], v_pages=g["v8"], k_scales=g["kz"], v_scales=g["vz"], page_table=g["table"], lengths=g["lengths"])

    def refused(error, **bad):
        args = dict(good, **bad)
        for call in (lambda: ops.paged_append_q8_(g["qkv"], 4, **args), lambda: ops.paged_attn_q8(g["q"], **args), lambda: ops.paged_read_q8(**args, places=20)):
            with pytest.raises(error):
                call()
    refused(ValueError, k_pages=torch.zeros_like(g["k8"], dtype=BF16), v_pages=torch.zeros_like(g["v8"], dtype=BF16))
    refused(ValueError, v_pages=g["v8"][:, :8])
    refused(ValueError, k_scales=g["kz"].view(torch.uint8))
    refused(ValueError, v_scales=g["vz"].float())
    refused(ValueError, k_scales=g["kz"][:-1], v_scales=g["vz"][:-1])
    refused(ValueError, k_scales=g["kz"][:, :, :1], v_scales=g["vz"][:, :, :1])
    refused(ValueError, k_scales=g["kz"][:, :0], v_scales=g["vz"][:, :0])
    refused(ValueError, v_scales=g["vz"][:, :1])
    refused(ValueError, page_table=g["table"].long())
    refused(ValueError, lengths=g["lengths"].long())
    refused(ValueError, lengths=g["lengths"][:1])
    refused(RuntimeError, k_scales=g["kz"].cpu(), v_scales=g["vz"].cpu())
    four = torch.zeros((g["k8"].shape[0], 4, 2), dtype=torch.uint8, device=dev).view(E8)
    with pytest.raises(_lib.OdysseusHipError, match="a scale for each 4 tokens"):
        ops.paged_attn_q8(g["q"], **dict(good, k_scales=four, v_scales=four))
    with pytest.raises(ValueError):
        ops.paged_append_q8_(g["qkv"], 3, **good)
    with pytest.raises(ValueError):
        ops.paged_append_q8_(g["qkv"], 4, **good, rotate=False, position_ids=torch.zeros((2, 1), dtype=torch.int64, device=dev))
    with pytest.raises(TypeError):
        ops.paged_attn_q8(g["q"].half(), **good)
    with pytest.raises(TypeError):
        ops.paged_read_q8(**good, places=5, dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.paged_read_q8(**good, places=-1)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.paged_attn_q8(g["q"].clone().requires_grad_(), **good)
