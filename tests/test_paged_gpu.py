"""A key / value cache in pages: appending with the rotation, attention over it, against 64 bits on the CPU."""
import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _to(c, dev):
    def move(t):   # keeps the strides: what is tested with a layout is that layout
        return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t)
    return {k: move(t) if torch.is_tensor(t) else t for k, t in c.items()}


def _inv_freq(D, base=10000.0):
    return 1.0 / (base ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D))


def _check_attn(c, g, scale=None):
    from odysseus_transformer_amd import ops
    out, lse = ops.paged_attn(g["q"], g["k"], g["v"], g["table"], g["lengths"], scale=scale, new_tokens=g.get("new"))
    torch.cuda.synchronize()
    o, s, mean, dots = ref.attend(c, scale)
    tol_o, tol_s = ref.attend_bounds(c, o, s, mean, dots)
    out, lse = out.double().cpu(), lse.double().cpu()
    none = s == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert (out[none.transpose(1, 2)] == 0).all()
    bad = (out - o).abs() > tol_o
    assert not bad.any(), f"out: {int(bad.sum())} of {bad.numel()} beyond their bounds, worst {((out - o).abs() / tol_o).max():.2f}"
    bad = ((lse - s).abs() > tol_s) & ~none
    assert not bad.any(), f"lse: {int(bad.sum())} beyond their bounds, worst {((lse - s).abs()[~none] / tol_s[~none]).max():.2f}"


def _check_append(c, g, Hq, positions=None, rotate=True):
    from odysseus_transformer_amd import ops
    D, dtype = c["q"].shape[3], c["q"].dtype
    f = _inv_freq(D)
    (q, q_size), (k, k_size), v = ref.append(c, Hq, f if rotate else None, positions)
    qkv = g["qkv"].clone()
    got = ops.paged_append_(g["qkv"], Hq, g["k"], g["v"], g["table"], g["lengths"],
                            position_ids=None if positions is None else positions.to(g["qkv"].device),
                            inv_freq=f.to(g["qkv"].device) if rotate else None, rotate=rotate, new_tokens=g.get("new"))
    torch.cuda.synchronize()
    assert torch.equal(g["qkv"], qkv), "the projection was written to"
    assert torch.equal(g["v"].cpu(), v.to(dtype)), "values"
    if not rotate:
        assert got.data_ptr() == g["qkv"].data_ptr() and torch.equal(got, g["qkv"][:, :, :Hq])
        assert torch.equal(g["k"].cpu(), k.to(dtype)), "keys"
        return
    half = torch.finfo(dtype).eps / 2
    for name, have, want, size in (("q", got, q, q_size), ("k", g["k"], k, k_size)):
        have = have.double().cpu()
        assert torch.equal(have[size == 0], want[size == 0]), f"{name}: rows without a new token"
        # one rounding of the result, the sum's in 32 bits, and a cosine within 2^-23 of the middle of two values of the type, which may round to either
        # one: a step of the type of one of the two products
        err = (have - want).abs()
        assert (err <= half * want.abs() + (2 * half + 2 ** -22) * size).all(), name
        # but hardly any of them do
        assert err.norm() <= (half + 2 ** -12 * half + 2 ** -22) * want.norm() + 2 * half * size.norm() * 2 ** -4, name
        tight = err <= half * want.abs() + 2 ** -21 * size
        assert tight.double().mean() > 0.998, f"{name}: {1 - tight.double().mean().item():.1e} of the values are further than their rounding"


APPEND = [
    # lengths, n, Hq, Hkv, D, page, dtype, layout
    ([1], 1, 1, 1, 128, 16, BF16, "rows"),
    ([5, 0, 17, 33, 8], 1, 4, 2, 128, 8, BF16, "rows"),            # a sequence that takes no part
    ([9, 3, 40], 9, 8, 2, 64, 16, BF16, "heads"),                  # padded on the left
    ([300, 131, 70], 67, 6, 3, 128, 32, BF16, "mixed"),
    ([100, 20], 33, 5, 1, 64, 64, F32, "rows"),
    ([41, 0, 1], 7, 4, 4, 128, 8, F32, "mixed"),
    ([2, 1], 2, 8, 8, 64, 256, F32, "heads"),
    ([700], 700, 4, 1, 128, 128, BF16, "rows"),
    (list(range(1, 98)), 1, 2, 1, 64, 16, BF16, "rows"),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "S%d_max%d_n%d_H%d_%d_D%d_p%d_%s_%s" % (len(c[0]), max(c[0]), *c[1:6], str(c[6])[-4:], c[7]))
def test_append(case, dev):
    lengths, n, Hq, Hkv, D, page, dtype, layout = case
    print(f"append {case}", flush=True)
    c = ref.make(lengths, n, Hq, Hkv, D, page, dtype, seed=n + Hq, layout=layout)
    _check_append(c, _to(c, dev), Hq)
    _check_append(c, _to(c, dev), Hq, rotate=False)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_append_with_positions_of_its_own(dtype, dev):
    """Positions apart from the places: far ones, whose angles are products of 32 bits, of each sequence and shared by all."""
    c = ref.make([50, 11, 30], 4, 4, 2, 128, 16, dtype, seed=3)
    own = torch.tensor([[131071, 0, 7, 99999], [1, 2, 3, 4], [65536, 65537, 12, 0]])
    _check_append(c, _to(c, dev), 4, positions=own)
    g = _to(c, dev)
    from odysseus_transformer_amd import ops
    shared = torch.tensor([3, 4, 5, 6], device=dev)
    a = ops.paged_append_(g["qkv"], 4, g["k"], g["v"], g["table"], g["lengths"], position_ids=shared)
    b = ops.paged_append_(g["qkv"], 4, g["k"], g["v"], g["table"], g["lengths"], position_ids=shared.to(torch.int32).expand(3, 4).contiguous())
    assert torch.equal(a, b)


def test_append_rotates_as_rope_does(dev):
    from odysseus_transformer_amd import ops
    for dtype in (BF16, F32):
        c = ref.make([77, 77], 77, 6, 2, 128, 16, dtype, seed=8)
        g = _to(c, dev)
        q = ops.paged_append_(g["qkv"], 6, g["k"], g["v"], g["table"], g["lengths"])
        x = g["qkv"].clone()
        ops.rope_(x, 8)
        assert torch.equal(q, x[:, :, :6])
        pages, rows = g["table"].long()[:, torch.arange(77) // 16], torch.arange(77, device=dev) % 16
        assert torch.equal(g["k"][pages, rows], x[:, :, 6:8])


ATTN = [
    # lengths, n, Hq, Hkv, D, page, dtype, layout
    ([1], 1, 1, 1, 128, 16, BF16, "rows"),
    ([1], 1, 1, 1, 64, 8, F32, "rows"),
    ([100], 1, 4, 1, 128, 16, BF16, "rows"),
    ([5, 0, 17, 33, 8, 128, 129, 127, 31, 32], 1, 4, 2, 128, 8, BF16, "rows"),
    ([700, 1, 64, 1029], 1, 8, 2, 64, 32, BF16, "heads"),
    ([2000, 513, 4], 1, 32, 8, 128, 64, BF16, "mixed"),
    ([600, 77], 1, 32, 1, 128, 16, BF16, "rows"),                 # 32 rows of one kv head
    ([600, 77], 1, 40, 1, 64, 16, BF16, "rows"),                  # 40
    ([400, 70], 1, 71, 1, 128, 16, BF16, "rows"),                 # 71
    ([300, 2], 5, 7, 1, 128, 16, BF16, "rows"),                   # 35 rows, padded on the left
    ([150, 40, 3, 0], 8, 8, 8, 64, 16, BF16, "heads"),
    ([333], 333, 4, 1, 128, 32, BF16, "rows"),                    # a whole prompt
    ([400, 90, 200], 130, 6, 2, 128, 64, BF16, "mixed"),
    ([260, 129], 65, 4, 4, 64, 8, BF16, "rows"),
    ([500, 33, 1, 0], 1, 8, 8, 64, 32, F32, "rows"),
    ([290, 40], 1, 24, 2, 128, 16, F32, "heads"),
    ([129, 64, 31], 6, 6, 2, 64, 8, F32, "mixed"),
    ([150, 20], 40, 4, 2, 128, 16, F32, "rows"),
    ([4096 + 3], 1, 8, 8, 128, 128, BF16, "rows"),
    ([3000], 1, 2, 2, 64, 256, F32, "rows"),
    (list(range(0, 260, 2)), 1, 2, 1, 64, 16, BF16, "rows"),      # more sequences than a wavefront has lanes
    ([8] * 300 + [900], 1, 2, 2, 64, 8, BF16, "rows"),
]
_ids = lambda c: "S%d_max%d_n%d_H%d_%d_D%d_p%d_%s_%s" % (len(c[0]), max(c[0]), *c[1:6], str(c[6])[-4:], c[7])  # noqa: E731


@pytest.mark.parametrize("case", ATTN, ids=_ids)
def test_attn(case, dev):
    lengths, n, Hq, Hkv, D, page, dtype, layout = case
    print(f"attn {case}", flush=True)
    c = ref.make(lengths, n, Hq, Hkv, D, page, dtype, seed=n + Hq + D, layout=layout)
    _check_attn(c, _to(c, dev))


def test_attn_scale_and_strided_queries(dev):
    c = ref.make([90, 200], 3, 4, 2, 128, 16, BF16, seed=1)
    g = _to(c, dev)
    for scale in (0.25, 0.0, -0.1):
        _check_attn(c, g, scale)
    c["q"] = c["qkv"][:, :, :4]
    g["q"] = g["qkv"][:, :, :4]                                   # a slice of the packed projection
    _check_attn(c, g)


NEW = [
    # lengths, new tokens, n, Hq, Hkv, D, page, dtype
    ([40, 300, 7, 90], [1, 1, 0, 1], 1, 8, 2, 128, 16, BF16),
    ([40, 300, 7, 90, 3], [5, 0, 2, 9, -1], 5, 4, 2, 64, 8, BF16),               # more than n, fewer than none
    ([150, 300, 100, 20], [64, 1, 0, 20], 64, 4, 1, 128, 32, BF16),              # tiles of a sequence without a token in front
    ([700, 150, 131, 60, 200], [130, 3, 0, 60, 129], 130, 4, 2, 128, 64, BF16),
    ([270, 90, 200], [1, 80, 66], 80, 2, 1, 64, 16, BF16),
    ([40, 300, 7, 90], [1, 0, 1, 0], 1, 4, 2, 64, 16, F32),
    ([90, 200, 33], [33, 2, 0], 33, 4, 1, 128, 8, F32),
    ([50, 60], [0, 0], 3, 4, 2, 128, 16, BF16),                                  # nobody
    ([500, 60], [0, 0], 100, 4, 2, 128, 16, BF16),
]


@pytest.mark.parametrize("case", NEW, ids=lambda c: "n%d_H%d_%d_D%d_p%d_%s" % (*c[2:7], str(c[7])[-4:]))
def test_sequences_with_fewer_new_tokens(case, dev):
    lengths, new, n, Hq, Hkv, D, page, dtype = case
    print(f"new {case}", flush=True)
    c = ref.make(lengths, n, Hq, Hkv, D, page, dtype, seed=n + D)
    c["new"] = torch.tensor(new, dtype=torch.int32)
    g = _to(c, dev)
    _check_attn(c, g)
    _check_append(c, g, Hq)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[64], [65, 1], [128, 63], [192, 191], [321, 448, 64], [130 + 64 * 9]], ids=str)
def test_chunks_of_few_tiles(D, lengths, dev):
    """As many tiles of keys as a loop with several of them in flight can begin and end with, n from one row more than the few-rows kernel takes."""
    for n in (65, 128, 200):
        c = ref.make(lengths, n, 2, 1, D, 8, BF16, seed=sum(lengths) + n)
        _check_attn(c, _to(c, dev))


@pytest.mark.parametrize("lengths", [[64], [65, 1], [128, 63], [192, 191], [256, 255], [321, 448, 64], [383], [577, 900], [1500]], ids=str)
def test_long_chunks_of_few_tiles(lengths, dev):
    """Pages of a tile of keys and more, tokens of one and of several tiles of 256 rows."""
    for n, Hq, page in ((129, 1, 64), (256, 2, 128), (70, 4, 64)):
        c = ref.make(lengths, n, Hq, 1, 128, page, BF16, seed=sum(lengths) + n)
        _check_attn(c, _to(c, dev))


@pytest.mark.parametrize("column", [0, 1, 4, 5, 8, 9, 10, 11])
def test_long_chunks_with_a_page_missing(column, dev):
    for new in (None, 150):
        c = ref.make([760, 90], 200, 4, 2, 128, 64, BF16, seed=column)
        c["table"][0, column] = 2 ** 31 - 1 if column % 2 else -1
        c["new"] = None if new is None else torch.tensor([new, 80], dtype=torch.int32)
        _check_attn(c, _to(c, dev))


def test_long_chunks_whose_scores_grow(dev):
    """The largest score of a row in every one of its tiles above those before it, by more and by less than a reference may lag behind."""
    for step in (0.5, 3.0, 40.0):
        c = ref.make([700], 140, 2, 1, 128, 64, BF16, seed=2)
        q = c["q"][0, 0, 0].float()
        for j in range(700):
            at = ref.page_of(c, 0, j)
            c["k"][at[0], at[1], 0] = (q * (step * (j // 32) / 20 * 11.3 / (q @ q).item() + 0.02 * torch.randn(128, generator=torch.Generator().manual_seed(j)))).to(BF16)
        c["q"][0, :, :] = q.to(BF16) * torch.linspace(-1, 1, 280).reshape(140, 2, 1).to(BF16)
        _check_attn(c, _to(c, dev))


def _sampled(c, g, count, seed):
    """_check_attn for some rows of a call that is too large for all of them, the first and the last one of each sequence's among them."""
    from odysseus_transformer_amd import ops
    out, lse = ops.paged_attn(g["q"], g["k"], g["v"], g["table"], g["lengths"], new_tokens=g.get("new"))
    out, lse = out.double().cpu(), lse.double().cpu()
    S, n, Hq = c["q"].shape[:3]
    Hkv = c["k"].shape[2]
    r = torch.Generator().manual_seed(seed)
    draw = lambda most: int(torch.randint(most, (1,), generator=r))  # noqa: E731
    rows = [(draw(S), draw(n), draw(Hq)) for _ in range(count)] + [(s, i, draw(Hq)) for s in range(min(S, 12)) for i in (0, n - 1)]
    for s, i, h in rows:
        kv = h * Hkv // Hq
        one = dict(c, q=c["q"][s:s + 1, i:i + 1, h:h + 1], k=c["k"][:, :, kv:kv + 1], v=c["v"][:, :, kv:kv + 1], table=c["table"][s:s + 1],
                   lengths=c["lengths"][s:s + 1] - n + i + 1, new=torch.tensor([int(i >= ref.first_token(c, s, n))]))
        o, z, mean, dots = ref.attend(one)
        tol_o, tol_s = ref.attend_bounds(one, o, z, mean, dots)
        if z.item() == -math.inf:
            assert lse[s, h, i] == -math.inf and (out[s, i, h] == 0).all(), (s, i, h)
            continue
        assert ((out[s, i, h] - o[0, 0, 0]).abs() <= tol_o[0, 0, 0]).all(), (s, i, h)
        assert (lse[s, h, i] - z[0, 0, 0]).abs() <= tol_s[0, 0, 0], (s, i, h)


# as many sequences and kv heads as tiles of 256 rows are taken for (heads of 64 in tiles of 128)
WIDE = [([64, 65, 128, 63, 192, 191, 256, 255], 200), ([321, 448, 200, 383, 577, 900, 260, 1500], 200), ([130] * 8, 250), ([700, 300, 257, 256, 1, 90, 0, 40], 256),
        ([33, 513, 769, 1025, 1281, 640, 704, 832], 512)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("lengths,n", WIDE, ids=lambda x: str(x) if isinstance(x, int) else "max%d" % max(x))
def test_tiles_of_256_rows(lengths, n, page, D, dev):
    """Ranges of one tile of keys to many, tokens and sequences that are not there, a page missing before, under and behind plain tiles."""
    for new, holes in ((False, False), (True, False), (False, True)):
        c = ref.make(lengths, n, 16 if n == 512 else 8, 8, D, page, BF16, seed=n + page)
        if new:
            c["new"] = torch.tensor([n, n // 2, 1, 0, n, 7, n, n - 1], dtype=torch.int32)
        if holes:
            for s, column in ((0, 0), (1, 3), (1, 200 // page), (5, 640 // page), (7, 1)):
                c["table"][s, min(column, c["table"].shape[1] - 1)] = -1 if s % 2 else 2 ** 31 - 1
        _sampled(c, _to(c, dev), 40, page)


@pytest.mark.parametrize("D", [64, 128])
def test_tiles_of_256_rows_whose_scores_grow(D, dev):
    """The largest score of a row in every one of its tiles above those before it, by more and by less than a reference may lag behind."""
    for step in (0.5, 3.0, 40.0):
        c = ref.make([700] * 8, 200, 8, 8, D, 64, BF16, seed=2)
        q = c["q"][0, 0, 0].float()
        for s in range(8):
            j = torch.arange(700)
            noise = torch.randn(700, D, generator=torch.Generator().manual_seed(s)) * 0.02
            k = (q * (step * (j // 32) / 20 * 11.3 / (q @ q).item())[:, None] + noise).to(BF16)
            c["k"][c["table"][s, j // 64].long(), j % 64] = k[:, None]
        c["q"][:] = q.to(BF16) * torch.linspace(-1, 1, 8 * 200 * 8).reshape(8, 200, 8, 1).to(BF16)
        _sampled(c, _to(c, dev), 60, 1)


@pytest.mark.parametrize("case", [([33000], 512, 32, 8, 64), ([33000], 512, 32, 8, 16), ([9000, 17000, 300], 300, 16, 8, 128),
                                  ([64 + 9 * i for i in range(70)], 64, 32, 8, 64), ([64 + 9 * i for i in range(70)], 64, 32, 8, 16),
                                  ([900 - 5 * i for i in range(170)], 1, 16, 4, 16), ([64 + 9 * i for i in range(70)], 10, 16, 4, 16),
                                  ([64 + 9 * i for i in range(20)], 40, 8, 8, 64)], ids=lambda c: "S%d_max%d_n%d_H%d_%d_p%d" % (len(c[0]), max(c[0]), *c[1:]))
def test_many_keys_and_many_sequences(case, dev):
    """More tiles for a block than pages are looked up at once; more units than blocks, each cut at most once."""
    lengths, n, Hq, Hkv, page = case
    c = ref.make(lengths, n, Hq, Hkv, 128, page, BF16, seed=n)
    _sampled(c, _to(c, dev), 30, 1)


@pytest.mark.parametrize("rows", [33, 47, 48, 49, 64, 65])
def test_rows_around_the_tiles(rows, dev):
    c = ref.make([500, 90, 33], rows, 2, 2, 128, 16, BF16, seed=rows)
    _check_attn(c, _to(c, dev))


@pytest.mark.parametrize("column", [0, 1, 5, 9, 10])
def test_chunks_with_a_page_missing(column, dev):
    """Tiles before and behind a missing page, which leaves holes in front of the newest tokens, under them, and at the start."""
    c = ref.make([352], 130, 4, 2, 128, 32, BF16, seed=column)
    c["table"][0, column] = -7
    _check_attn(c, _to(c, dev))


def test_both_host_paths_agree(dev, monkeypatch):
    from odysseus_transformer_amd import ops
    c = ref.make([300, 40, 9], 3, 8, 2, 128, 16, BF16, seed=14)
    c["new"] = torch.tensor([3, 1, 0], dtype=torch.int32)
    res = []
    for native in (True, False):
        if not native:
            for name in ("paged_append", "paged_attn"):
                monkeypatch.setattr(ops.native, name, lambda *a: None)
        g = _to(c, dev)
        q = ops.paged_append_(g["qkv"], 8, g["k"], g["v"], g["table"], g["lengths"], new_tokens=g["new"])
        own = ops.paged_append_(g["qkv"], 8, g["k"], g["v"], g["table"], g["lengths"], position_ids=torch.arange(3, device=dev), base=500.0)
        held = ops.paged_append_(g["qkv"], 8, g["k"], g["v"], g["table"], g["lengths"], rotate=False, new_tokens=g["new"])
        assert held.data_ptr() == g["qkv"].data_ptr()
        res.append((q, own, held, g["k"], g["v"], *ops.paged_attn(q, g["k"], g["v"], g["table"], g["lengths"], new_tokens=g["new"]),
                    *ops.paged_attn(q, g["k"], g["v"], g["table"], g["lengths"], 0.3)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_unowned_rows_are_neither_read_nor_written(dev):
    """NaN in every row that belongs to no token, the tail of the last pages among them."""
    from odysseus_transformer_amd import ops
    c = ref.make([37, 5, 130], 1, 4, 2, 128, 16, BF16, seed=2)
    owned = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for s, length in enumerate(c["lengths"].tolist()):
        for j in range(length):
            owned[ref.page_of(c, s, j)] = True
    for t in ("k", "v"):
        c[t][~owned] = float("nan")
    g = _to(c, dev)
    _check_attn(c, g)
    ops.paged_append_(g["qkv"], 4, g["k"], g["v"], g["table"], g["lengths"])
    for t in ("k", "v"):
        now = g[t].cpu()
        assert now[~owned].isnan().all()
        assert torch.isfinite(now[owned]).all()


@pytest.mark.parametrize("n", [1, 3, 70])
def test_entries_that_are_no_page(n, dev):
    """Table entries outside the pool (below, at its end, far behind): their places hold nothing and nothing is written or read there;
    lengths behind the last column and below zero likewise."""
    c = ref.make([200, 100, 100, 64, 90], n, 4, 2, 64, 16, BF16, seed=5)
    pages = c["k"].shape[0]
    c["table"][0, 3] = -1
    c["table"][0, 12] = pages                                     # the newest tokens'
    c["table"][1, 0] = 2 ** 31 - 1
    c["table"][2, :] = -2 ** 31
    c["lengths"][3] = 2 ** 31 - 1                                 # far beyond what the table can hold
    c["lengths"][4] = -2 ** 31
    c["table"][3, 4:] = -1
    if n == 1:
        c["table"][3, 5] = c["table"][3, 1]
    g = _to(c, dev)
    full = dict(c, lengths=c["lengths"].clone())
    # in 64 bits a length of 2^31 - 1 is walked by its columns only: all places of the table are before every new token
    full["lengths"][3] = c["table"].shape[1] * 16 + n
    _check_attn(full, g)
    c2 = dict(full)
    from odysseus_transformer_amd import ops
    before = g["k"].clone(), g["v"].clone()
    f = _inv_freq(64)
    (q, q_size), (k, k_size), v = ref.append(c2, 4, f)
    got = ops.paged_append_(g["qkv"], 4, g["k"], g["v"], g["table"], g["lengths"], inv_freq=f.to(dev))
    assert torch.equal(g["v"].cpu(), v.to(BF16))
    untouched = k_size == 0
    assert torch.equal(g["k"].cpu()[untouched], before[0].cpu()[untouched])
    assert (got[4] == 0).all() and torch.isfinite(got).all()


def test_sequences_that_share_pages(dev):
    c = ref.make([80, 80, 80], 1, 4, 2, 128, 16, BF16, seed=6)
    c["table"][1, :4] = c["table"][0, :4]
    c["table"][2, :5] = c["table"][0, 0]                          # one page five times
    _check_attn(c, _to(c, dev))


def test_infinite_and_nan_values_reach_their_own_sequence_only(dev):
    from odysseus_transformer_amd import ops
    c = ref.make([60, 60, 60, 60], 1, 4, 2, 128, 16, BF16, seed=7)
    g = _to(c, dev)
    clean, clean_lse = ops.paged_attn(g["q"], g["k"], g["v"], g["table"], g["lengths"])
    g["k"][int(c["table"][1, 1]), 3, 0] = float("nan")            # kv head 0: query heads 0, 1
    g["v"][int(c["table"][2, 2]), 1, 1] = float("inf")
    out, lse = ops.paged_attn(g["q"], g["k"], g["v"], g["table"], g["lengths"])
    assert out[1, 0, :2].isnan().all() and lse[1, :2].isnan().all()
    assert torch.equal(out[1, 0, 2:], clean[1, 0, 2:])
    assert (out[2, 0, 2:] == float("inf")).all() and torch.equal(lse[2], clean_lse[2]) and torch.equal(out[2, 0, :2], clean[2, 0, :2])
    for s in (0, 3):
        assert torch.equal(out[s], clean[s]) and torch.equal(lse[s], clean_lse[s])


def test_large_scores(dev):
    """Scores far apart, the largest last and first: no sum overflows or vanishes."""
    for at in (0, 250, 299):
        c = ref.make([300], 1, 2, 1, 64, 16, BF16, seed=9)
        c["k"] *= 4
        place = ref.page_of(c, 0, at)
        c["k"][place] = c["q"][0, 0, 0] * 6
        _check_attn(c, _to(c, dev))


def test_offsets_beyond_32_bits(dev):
    """Pages whose elements lie more than 2^31 from the pool's start."""
    pages, page, Hkv, D = 17000, 128, 8, 128                       # 2.2e9 elements
    from odysseus_transformer_amd import ops
    k = torch.zeros((pages, page, Hkv, D), dtype=BF16, device=dev)
    v = torch.zeros((pages, page, Hkv, D), dtype=BF16, device=dev)
    ids = [0, 16999, 16500, 3]
    table = torch.tensor([ids], dtype=torch.int32, device=dev)
    small = ref.make([400], 1, 16, Hkv, D, page, BF16, seed=11)
    for c, p in enumerate(ids):
        k[p].copy_(small["k"][int(small["table"][0, c])])
        v[p].copy_(small["v"][int(small["table"][0, c])])
    lengths = torch.tensor([400], dtype=torch.int32, device=dev)
    g = _to(small, dev)
    for n in (1, 40):
        q = torch.randn((1, n, 16, D), device=dev).to(BF16)
        want = ops.paged_attn(q, g["k"], g["v"], g["table"], g["lengths"])
        got = ops.paged_attn(q, k, v, table, lengths)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lengths += 20                                                  # into page 3 from place 384 on
    qkv = torch.randn((1, 200, 32, D), device=dev).to(BF16)
    ops.paged_append_(qkv, 16, k, v, table, lengths, rotate=False)
    rows = torch.arange(220, 420, device=dev)
    at = (torch.tensor(ids, device=dev)[rows // page], rows % page)
    assert torch.equal(v[at], qkv[0, :, 24:]) and torch.equal(k[at], qkv[0, :, 16:24])


def test_attends_what_was_appended_step_by_step(dev):
    """A prompt, then single tokens, against attention over the whole sequence at once."""
    from odysseus_transformer_amd import ops
    L0, steps, Hq, Hkv, D, page = 45, 23, 8, 2, 128, 16
    for dtype in (BF16, F32):
        x = torch.randn((1, L0 + steps, Hq + 2 * Hkv, D), generator=torch.Generator().manual_seed(4)).to(dtype).to(dev)
        whole = x.clone()
        ops.rope_(whole, Hq + Hkv)
        want, want_lse = ops.attn_fwd(whole[:, :, :Hq], whole[:, :, Hq:Hq + Hkv], whole[:, :, Hq + Hkv:], causal=True)
        k, v = (torch.full((7, page, Hkv, D), float("nan"), dtype=dtype, device=dev) for _ in range(2))
        table = torch.tensor([[4, 0, 6, 2, 5]], dtype=torch.int32, device=dev)
        lengths = torch.zeros(1, dtype=torch.int32, device=dev)
        out, lse = [], []
        for a, b in [(0, L0)] + [(t, t + 1) for t in range(L0, L0 + steps)]:
            lengths += b - a
            q = ops.paged_append_(x[:, a:b], Hq, k, v, table, lengths)
            o, s = ops.paged_attn(q, k, v, table, lengths)
            out.append(o)
            lse.append(s)
        out, lse = torch.cat(out, 1), torch.cat(lse, 2)
        # both round p and the result once: twice the bound of one
        half = torch.finfo(dtype).eps / 2
        bound = 2 * (2 * half + 1e-5) * whole[:, :, Hq + Hkv:].float().abs().amax()
        assert (out.float() - want.float()).abs().max() <= bound
        assert (lse - want_lse).abs().max() <= 1e-4


def test_replayed_from_a_graph_with_other_lengths_and_pages(dev):
    """A decoding step as a captured graph: appended to and attended with whatever table and lengths hold at the replay; two graphs that
    take turns, eager calls between them."""
    from odysseus_transformer_amd import ops
    Hq, Hkv, D, page = 8, 2, 128, 16
    base = ref.make([40, 3, 0, 90], 1, Hq, Hkv, D, page, BF16, seed=12)
    wide = ref.make([40] * 40, 1, Hq, Hkv, D, page, BF16, seed=13)
    sets, graphs = [_to(base, dev), _to(wide, dev)], []

    def step(g):
        q = ops.paged_append_(g["qkv"], Hq, g["k"], g["v"], g["table"], g["lengths"])
        return ops.paged_attn(q, g["k"], g["v"], g["table"], g["lengths"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for g in sets:
            step(g)
    torch.cuda.current_stream().wait_stream(side)
    for g in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(g)
        graphs.append((graph, res))
    for turn in range(3):
        for g, (graph, res) in zip(sets, graphs):
            g["lengths"].copy_((g["lengths"] + 1) * (g["lengths"] > 0))
            g["qkv"].normal_()
            pools = g["k"].clone(), g["v"].clone()
            graph.replay()
            torch.cuda.synchronize()
            got = res[0].clone(), res[1].clone(), g["k"].clone(), g["v"].clone()
            g["k"].copy_(pools[0])
            g["v"].copy_(pools[1])
            want = step(g)
            for a, b in zip(got, (*want, g["k"], g["v"])):
                assert torch.equal(a, b), f"turn {turn}"


def test_calls_on_two_streams_at_once(dev):
    from odysseus_transformer_amd import ops
    cs = [_to(ref.make([900, 30, 411], 1, 16, 4, 128, 32, BF16, seed=20 + i), dev) for i in range(2)]
    want = [ops.paged_attn(c["q"], c["k"], c["v"], c["table"], c["lengths"]) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, cs)):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attn(c["q"], c["k"], c["v"], c["table"], c["lengths"]))
    torch.cuda.synchronize()
    for i in range(2):
        for o, s in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(s, want[i][1])


def test_nothing_to_do(dev):
    from odysseus_transformer_amd import ops
    c = _to(ref.make([5, 6], 1, 4, 2, 64, 8, BF16, seed=1), dev)
    q = ops.paged_append_(c["qkv"][:, :0], 4, c["k"], c["v"], c["table"], c["lengths"])
    assert q.shape == (2, 0, 4, 64)
    out, lse = ops.paged_attn(c["q"][:0], c["k"], c["v"], c["table"][:0], c["lengths"][:0])
    assert out.shape == (0, 1, 4, 64) and lse.shape == (0, 4, 1)


def test_refusals(dev):
    from odysseus_transformer_amd import ops
    from odysseus_transformer_amd._lib import OdysseusHipError
    c = _to(ref.make([5, 6], 1, 4, 2, 64, 8, BF16, seed=1), dev)
    args = lambda **kw: [{**c, **kw}[k] for k in ("k", "v", "table", "lengths")]  # noqa: E731
    for kw in (dict(k=c["k"].float()), dict(v=c["v"][:, :, :1]), dict(table=c["table"].long()), dict(table=c["table"][:1]), dict(table=c["table"].t().contiguous().t()),
               dict(lengths=c["lengths"].long()), dict(lengths=c["lengths"][:1]), dict(k=c["k"].transpose(2, 3), v=c["v"].transpose(2, 3))):
        with pytest.raises(ValueError):
            ops.paged_attn(c["q"], *args(**kw))
        with pytest.raises(ValueError):
            ops.paged_append_(c["qkv"], 4, *args(**kw))
    with pytest.raises(ValueError):
        ops.paged_append_(c["qkv"], 3, *args())
    with pytest.raises(ValueError):
        ops.paged_append_(c["qkv"], 4, *args(), position_ids=torch.zeros((2, 3), dtype=torch.int64, device=dev))
    with pytest.raises(TypeError):
        ops.paged_attn(c["q"].half(), c["k"].half(), c["v"].half(), c["table"], c["lengths"])
    with pytest.raises(OdysseusHipError):          # 3 heads on 2
        ops.paged_attn(c["q"][:, :, :3], *args())
    with pytest.raises(OdysseusHipError):          # a page of 5 rows
        ops.paged_attn(c["q"], *args(k=c["k"][:, :5], v=c["v"][:, :5]))
    with pytest.raises(OdysseusHipError):          # a row that does not start on 16 bytes
        flat = torch.zeros(c["q"].numel() + 1, dtype=BF16, device=dev)
        ops.paged_attn(flat[1:].view(c["q"].shape), *args())
    with pytest.raises(RuntimeError):
        ops.paged_attn(c["q"].clone().requires_grad_(True), *args())
    with torch.no_grad():
        ops.paged_attn(c["q"].clone().requires_grad_(True), *args())
    with pytest.raises(RuntimeError):
        ops.paged_attn(c["q"].cpu(), *args())


# ---------------------------------------------------------------- the cache under the attention module and the decoder layer
def _config(d, Hq, Hkv, D, inter=512):
    import types
    return types.SimpleNamespace(hidden_size=d, num_attention_heads=Hq, num_key_value_heads=Hkv, head_dim=D, intermediate_size=inter, hidden_act="silu",
                                 attention_dropout=0.0, rms_norm_eps=1e-6, rope_theta=10000.0, pretraining_tp=1)


def _layer(dtype, D, dev, **kw):
    from odysseus_transformer_amd.decoder.odysseus import OdysseusDecoderLayer
    torch.manual_seed(3)
    layer = OdysseusDecoderLayer(_config(256, 4, 2, D), **kw).to(dtype).to(dev).eval()
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(torch.randn(p.shape, dtype=torch.float32).to(p) * 0.05 if p.dim() > 1 else 1 + 0.1 * torch.randn(p.shape, dtype=torch.float32).to(p))
    return layer


def _cache(dtype, D, dev, **kw):
    from odysseus_transformer_amd.utils.paged_cache import PagedKVCache
    c = PagedKVCache(**{**dict(num_layers=1, num_pages=40, max_sequences=3, max_length=200, n_kv_heads=2, head_dim=D, page_size=16, dtype=dtype, device=dev), **kw})
    for t in c.layer(0):
        t.fill_(float("nan"))                                     # nothing that was not written may be read
    return c


def _whole(layer, x):
    """The layer over a whole sequence at once, in float32 on the CPU, by the formulas."""
    import odysseus_oracle as o
    a, m = layer.self_attn, layer.mlp
    f = lambda t: t.detach().float().cpu()  # noqa: E731
    norm = lambda h, w: h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * f(w)  # noqa: E731
    w = f(a.qkv_proj.weight) if a.pack_weight else torch.cat([f(t.weight) for t in (a.q_proj, a.k_proj, a.v_proj)])
    x = f(x)
    n = norm(x, layer.input_layernorm.weight)
    h = x + torch.cat([o.attention_block(r[None], w, f(a.o_proj.weight), a.num_heads, a.num_key_value_heads, a.head_dim)[0] for r in n])
    n = norm(h, layer.post_attention_layernorm.weight)
    gate, up = (n @ f(m.gate_up_proj.weight).t()).chunk(2, -1)
    return h + (torch.nn.functional.silu(gate) * up) @ f(m.down_proj.weight).t()


def _tol(dtype, steps=12):
    """Relative to a row's norm: so many roundings to the type on the way, half a step each, and sums of up to 512 products on both sides."""
    return steps * torch.finfo(dtype).eps / 2 + 1024 * 2 ** -24


@pytest.mark.parametrize("dtype,D,kw", [(BF16, 128, {}), (BF16, 64, {}), (BF16, 128, dict(fused=False)), (F32, 64, {})], ids=["bf16_128", "bf16_64", "plain", "f32"])
def test_decoder_layer_over_a_cache_in_pages(dtype, D, kw, dev):
    """Prompts of different lengths, single tokens, a step for some only, proposed tokens that are taken back, a sequence that ends and one that begins in
    its place: every row is the one that the layer gives for the whole sequence at once."""
    layer, cache = _layer(dtype, D, dev, **kw), _cache(dtype, D, dev)
    g = torch.Generator().manual_seed(5)
    rows = [torch.randn(1, 200, 256, generator=g).to(dtype) for _ in range(4)]
    want = [_whole(layer, r) for r in rows]
    row_of, at = [0, 1, 2], [0, 0, 0]

    def step(new):
        n = cache.begin(new)
        x = torch.zeros(3, n, 256, dtype=dtype)
        for s, t in enumerate(new):
            x[s, n - t:] = rows[row_of[s]][0, at[s]:at[s] + t]
        with torch.no_grad():
            y = layer(x.to(dev), past_key_values=cache)
        for s, t in enumerate(new):
            r, e = want[row_of[s]][0, at[s]:at[s] + t], y[s, n - t:].float().cpu()
            assert y[s, n - t:].isfinite().all()
            assert (e - r).norm() <= _tol(dtype) * r.norm(), f"step {new}, sequence {s}: {(e - r).norm() / r.norm():.2e}"
            at[s] += t
        assert y.isfinite().all()

    step([70, 9, 33])
    for _ in range(3):
        step([1, 1, 1])
    step([1, 0, 1])
    step([0, 20, 1])
    step([66, 5, 2])
    at[0] -= 40
    cache.truncate(0, at[0])
    step([40, 1, 1])
    cache.free(1)
    row_of[1], at[1] = 3, 0
    step([1, 50, 0])
    step([1, 1, 1])


def test_equal_prompts_into_an_empty_cache(dev):
    """Where a cache holds nothing else, attention reads the tokens at hand: what it holds afterwards serves the next steps."""
    for dtype, D in ((BF16, 128), (BF16, 64), (F32, 128)):
        layer = _layer(dtype, D, dev)
        x = torch.randn(3, 61, 256, generator=torch.Generator().manual_seed(6)).to(dtype).to(dev)
        a, b = _cache(dtype, D, dev), _cache(dtype, D, dev)
        want = _whole(layer, x)
        with torch.no_grad():
            a.begin([60, 60, 60])
            b.begin([60, 60, 60])
            assert a.fresh and b.fresh
            b.fresh = False
            ya, yb = layer(x[:, :60], past_key_values=a), layer(x[:, :60], past_key_values=b)
            for y in (ya, yb):
                assert (y.float().cpu() - want[:, :60]).norm() <= _tol(dtype) * want[:, :60].norm()
            for c in (a, b):
                c.begin(1)
                y = layer(x[:, 60:], past_key_values=c)
                assert (y.float().cpu() - want[:, 60:]).norm() <= _tol(dtype) * want[:, 60:].norm()


def test_unpacked_projections_and_a_lone_sequence(dev):
    from odysseus_transformer_amd.decoder.odysseus import LlamaFlashAttention2TPSP
    import odysseus_oracle as o
    for D in (64, 128):
        torch.manual_seed(4)
        m = LlamaFlashAttention2TPSP(_config(256, 4, 2, D), 0, pack_weight=False).to(BF16).to(dev).eval()
        f = lambda t: t.weight.detach().float().cpu()  # noqa: E731
        x = torch.randn(1, 44, 256).to(BF16)
        want = o.attention_block(x.float(), torch.cat((f(m.q_proj), f(m.k_proj), f(m.v_proj))), f(m.o_proj), 4, 2, D)[0]
        cache, at = _cache(BF16, D, dev, max_sequences=1), 0
        for n in (40, 1, 3):
            cache.begin([n])
            with torch.no_grad():
                y, _, c = m(x[:, at:at + n].to(dev), past_key_value=cache)
            assert c is cache
            r = want[:, at:at + n]
            assert (y.float().cpu() - r).norm() <= _tol(BF16, 8) * r.norm()
            at += n


def test_captured_step_of_a_layer_is_replayed_behind_begin(dev):
    """A decoding step as a graph: begin() rewrites what it reads.  Three and four sequences: norms in the products' prologues and apart."""
    for S in (3, 6):
        layer = _layer(BF16, 128, dev)
        caches = [_cache(BF16, 128, dev, max_sequences=S, num_pages=80) for _ in range(2)]
        x = torch.randn(S, 60, 256, generator=torch.Generator().manual_seed(8)).to(BF16).to(dev)
        first = [20, 3, 31, 1, 8, 16][:S]
        for c in caches:
            n = c.begin(first)
            with torch.no_grad():
                layer(x[:, :n], past_key_values=c)
        static = torch.zeros(S, 1, 256, dtype=BF16, device=dev)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        caches[0].begin(1)
        with torch.no_grad():
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                layer(static, past_key_values=caches[0])
            torch.cuda.current_stream().wait_stream(side)
            with torch.cuda.graph(graph):
                y = layer(static, past_key_values=caches[0])
        for s in range(S):
            caches[0].truncate(s, first[s])                       # the rehearsal's token
        for t in range(6):
            new = [1] * S if t != 3 else [1, 0] + [1] * (S - 2)
            static.copy_(x[:, 40 + t:41 + t])
            caches[0].begin(new)
            graph.replay()
            got = y.clone()
            caches[1].begin(new)
            with torch.no_grad():
                want = layer(static, past_key_values=caches[1])
            live = torch.tensor(new, device=dev) > 0
            assert torch.equal(got[live], want[live]), f"step {t}"
        # a step into an empty cache, captured: not one that a later replay may take for the first
        cache = _cache(BF16, 128, dev, max_sequences=S, num_pages=80)
        one, y1 = torch.cuda.CUDAGraph(), None
        cache.begin([1] * S)
        assert cache.fresh
        with torch.no_grad(), torch.cuda.graph(one):
            y1 = layer(static, past_key_values=cache)
        for s in range(S):
            cache.truncate(s, 0)
            caches[1].free(s)
        for t in range(3):
            static.copy_(x[:, t:t + 1])
            for c in (cache, caches[1]):
                c.begin([1] * S)
            one.replay()
            with torch.no_grad():
                want = layer(static, past_key_values=caches[1])
            err = (y1.float() - want.float()).norm() / want.float().norm()
            assert err <= _tol(BF16, 24), f"step {t}: {err:.2e}"    # the eager one's first step reads the tokens at hand


def test_module_refuses_gradients_through_the_cache(dev):
    layer, cache = _layer(BF16, 64, dev), _cache(BF16, 64, dev)
    cache.begin([3, 3, 0])
    x = torch.zeros(3, 3, 256, dtype=BF16, device=dev)
    with pytest.raises(RuntimeError, match="backward"):
        layer(x, past_key_values=cache)                           # the weights want gradients
    with torch.no_grad():
        layer(x, past_key_values=cache)
        with pytest.raises(ValueError, match="bfloat16|float32"):
            layer(x, past_key_values=_begun(_cache(F32, 64, dev)))


def test_book_keeping_is_not_captured(dev):
    cache = _cache(BF16, 64, dev)
    cache.begin([5, 3])
    before = cache.page_table.clone(), cache.sequence_lengths(), cache.free_pages()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device=dev)
    with torch.cuda.graph(graph):
        y = x + 1
        for call in (lambda: cache.begin(1), lambda: cache.truncate(0, 2), lambda: cache.free(1)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    graph.replay()
    assert (y == 1).all() and torch.equal(cache.page_table, before[0]) and cache.sequence_lengths() == before[1] and cache.free_pages() == before[2]
    cache.begin(1)


def _begun(cache):
    cache.begin([3, 3, 0])
    return cache


@pytest.mark.parametrize("fuse_layers", [False, True], ids=["modules_swapped", "layers_swapped"])
def test_host_model_decodes_with_a_cache_in_pages(fuse_layers, dev):
    """A patched host model: prompts of different lengths, then greedy tokens, against the oracle's layers over each sequence alone."""
    transformers = pytest.importorskip("transformers")
    import odysseus_oracle as o
    from odysseus_transformer_amd.decoder.odysseus import apply_odysseus_attn_patch_llama
    cfg = transformers.LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                   vocab_size=300, max_position_embeddings=512, rms_norm_eps=1e-6)
    torch.manual_seed(9)
    model = transformers.LlamaForCausalLM(cfg).float()
    apply_odysseus_attn_patch_llama(model, fuse_layers=fuse_layers)
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(torch.randn(p.shape) * 0.05 if p.dim() > 1 else 1 + 0.1 * torch.randn(p.shape))
    model = model.eval().to(dev)
    sd = {k: v.float().cpu() for k, v in model.state_dict().items()}

    def alone(seq):
        h = sd["model.embed_tokens.weight"][torch.tensor([seq])]
        for i in range(2):
            at = f"model.layers.{i}."
            h = o.decoder_layer_fwd(h, {name: sd[at + key] for name, key in (
                ("ln1", "input_layernorm.weight"), ("w_qkv", "self_attn.qkv_proj.weight"), ("w_o", "self_attn.o_proj.weight"),
                ("ln2", "post_attention_layernorm.weight"), ("w_gate_up", "mlp.gate_up_proj.weight"), ("w_down", "mlp.down_proj.weight"))}, 4, 2, 64)
        return o.linear_fwd(o.rmsnorm(h, sd["model.norm.weight"]), sd["lm_head.weight"])[0, -1]

    seqs = [torch.randint(0, 300, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (40, 13, 27)]
    cache = _cache(F32, 64, dev, num_layers=2)
    for t in cache.layer(1):
        t.fill_(float("nan"))
    n = cache.begin([len(q) for q in seqs])
    ids = torch.tensor([[0] * (n - len(q)) + q for q in seqs], device=dev)
    for _ in range(6):
        with torch.no_grad():
            logits = model(ids, past_key_values=cache, use_cache=True).logits[:, -1].cpu()
        for s, q in enumerate(seqs):
            want = alone(q)
            assert (logits[s] - want).norm() <= 2 * _tol(F32) * want.norm(), s    # two layers
            q.append(int(want.argmax()))
        cache.begin(1)
        ids = torch.tensor([q[-1:] for q in seqs], device=dev)
