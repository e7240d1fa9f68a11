"""A key / value cache in pages on the kernels that calls of other sizes take: many heads and many tokens to append, tables that are wider than any sequence,
chunks in tiles of 128 and of 256 rows with content, scales, graphs and streams of every kind."""
import math

import pytest
import torch

import paged_reference as ref
from test_paged_gpu import BF16, F32, _check_append, _check_attn, _to

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ appending
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(32, 8, 128, BF16), (32, 32, 64, BF16), (33, 11, 128, BF16), (32, 8, 128, F32), (15, 1, 128, F32), (64, 8, 64, F32)],
                         ids=lambda x: str(x)[-4:])
def test_append_of_more_heads_than_a_block_takes_at_once(Hq, Hkv, D, dtype, dev):
    """More than 256 pairs of vectors a token: a thread's second one and further ones."""
    c = ref.make([40, 3, 0, 17], 5, Hq, Hkv, D, 16, dtype, seed=Hq)
    _check_append(c, _to(c, dev), Hq)
    _check_append(c, _to(c, dev), Hq, rotate=False)


@pytest.mark.parametrize("rotate", [True, False], ids=["rotated", "as_it_is"])
@pytest.mark.parametrize("dtype,D,Hq,Hkv", [(BF16, 128, 32, 8), (BF16, 64, 32, 32), (F32, 128, 32, 8), (F32, 64, 16, 8)], ids=lambda x: str(x)[-4:])
def test_append_of_more_than_the_last_level_cache_holds(dtype, D, Hq, Hkv, rotate, dev):
    """More than 192 MiB read and written: padding, missing pages and unowned rows among them."""
    size = torch.finfo(dtype).bits // 8
    n = (192 << 20) // (2 * 3 * (Hq + 2 * Hkv) * D * size) + 2
    c = ref.make([n + 33, n, n - 500], n, Hq, Hkv, D, 64, dtype, seed=D)
    c["table"][1, 5] = -1
    assert 2 * c["qkv"].numel() * size > 192 << 20
    g = _to(c, dev)
    _check_append(c, g, Hq, rotate=rotate)


# ------------------------------------------------------------------------------------------------ attention
def _rows(c, g, count, seed, scale=None, got=None):
    """Some rows of a call against 64 bits, the first and the last one of each sequence's among them."""
    from odysseus_transformer_amd import ops
    out, lse = got or ops.paged_attn(g["q"], g["k"], g["v"], g["table"], g["lengths"], scale, new_tokens=g.get("new"))
    out, lse = out.double().cpu(), lse.double().cpu()
    S, n, Hq = c["q"].shape[:3]
    Hkv = c["k"].shape[2]
    r = torch.Generator().manual_seed(seed)
    draw = lambda most: int(torch.randint(most, (1,), generator=r))  # noqa: E731
    for s, i, h in [(draw(S), draw(n), draw(Hq)) for _ in range(count)] + [(s, i, draw(Hq)) for s in range(min(S, 12)) for i in (0, n - 1)]:
        kv = h * Hkv // Hq
        one = dict(c, q=c["q"][s:s + 1, i:i + 1, h:h + 1], k=c["k"][:, :, kv:kv + 1], v=c["v"][:, :, kv:kv + 1], table=c["table"][s:s + 1],
                   lengths=c["lengths"][s:s + 1] - n + i + 1, new=torch.tensor([int(i >= ref.first_token(c, s, n))]))
        o, z, mean, dots = ref.attend(one, scale)
        tol_o, tol_s = ref.attend_bounds(one, o, z, mean, dots)
        if z.item() == -math.inf:
            assert lse[s, h, i] == -math.inf and (out[s, i, h] == 0).all(), (s, i, h)
            continue
        assert ((out[s, i, h] - o[0, 0, 0]).abs() <= tol_o[0, 0, 0]).all(), (s, i, h)
        assert (lse[s, h, i] - z[0, 0, 0]).abs() <= tol_s[0, 0, 0], (s, i, h)
    return out, lse


def _widen(c, columns, seed):
    """The table with so many columns behind those in use, which hold pages of others: no place in them has a token."""
    S, width = c["table"].shape
    more = torch.randint(c["k"].shape[0], (S, columns), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    return dict(c, table=torch.cat((c["table"], more), 1))


WIDER = [
    # lengths, n, Hq, Hkv, D, page, dtype, columns
    ([100], 1, 32, 8, 128, 16, BF16, 505),                        # what a cache for 8192 tokens hands over
    ([1], 1, 4, 1, 128, 64, BF16, 2048),
    ([100, 0, 129, 700], 1, 32, 8, 128, 16, BF16, 505),
    ([100, 64, 33], 1, 8, 4, 64, 16, F32, 300),
    ([130, 20], 5, 8, 2, 64, 32, BF16, 200),
    ([500], 17, 16, 4, 128, 16, BF16, 2000),                      # 68 rows: in tiles of 128 for more than 16384 places
    ([500], 17, 16, 4, 128, 16, BF16, 500),                       # ... of 32 for fewer
    ([40, 9], 12, 16, 2, 64, 16, F32, 400),
    ([150, 90, 1], 130, 4, 2, 128, 64, BF16, 600),
    ([200, 130, 140, 150, 160, 170, 100, 190], 100, 16, 8, 128, 16, BF16, 900),   # in tiles of 256
    ([100] * 70, 1, 4, 2, 128, 16, BF16, 505),
]


@pytest.mark.parametrize("case", WIDER, ids=lambda c: "S%d_max%d_n%d_H%d_%d_D%d_p%d_%s_%d" % (len(c[0]), max(c[0]), *c[1:6], str(c[6])[-4:], c[7]))
def test_tables_wider_than_any_sequence(case, dev):
    """Ranges and their join by the table's width, keys of one or few of them."""
    lengths, n, Hq, Hkv, D, page, dtype, columns = case
    c = ref.make(lengths, n, Hq, Hkv, D, page, dtype, seed=n + D)
    c = _widen(c, columns, n)
    g = _to(c, dev)
    if len(lengths) * n * Hq > 1000:
        _rows(c, g, 40, n)
    else:
        _check_attn(c, g)


# lengths, n, Hq, Hkv, D, page.  From 64 (sequence, row tile, kv head) on heads of 128 run in tiles of 256 rows, others in tiles of 128
MANY_ROWS = {
    "wide_p64": ([700, 300, 257, 256, 1, 90, 0, 1041], 200, 8, 8, 128, 64),
    "wide_p16": ([700, 300, 257, 256, 1, 90, 0, 1041], 200, 8, 8, 128, 16),
    "chunk": ([700, 300, 1], 200, 8, 2, 128, 16),
    "chunk_D64": ([700, 300, 1, 513], 130, 8, 4, 64, 32),
    "lone": ([2100], 150, 2, 1, 128, 64),                         # cut over many blocks
}


@pytest.fixture(params=MANY_ROWS, scope="module")
def many_rows(request):
    return MANY_ROWS[request.param]


@pytest.mark.parametrize("name", MANY_ROWS)
def test_kernels_of_these_sizes(name, dev):
    """What the sizes below are for: the kernel that they run on."""
    from conftest import device_kernels
    from odysseus_transformer_amd import ops
    lengths, n, Hq, Hkv, D, page = MANY_ROWS[name]
    g = _to(ref.make(lengths, n, Hq, Hkv, D, page, BF16, seed=1), dev)
    _, kernels = device_kernels(lambda: ops.paged_attn(g["q"], g["k"], g["v"], g["table"], g["lengths"]))
    wanted = "paged_wide_kernel" if name.startswith("wide") else "paged_chunk_kernel"
    assert any(wanted in k for k in kernels), kernels


@pytest.mark.parametrize("holes", [False, True], ids=["whole", "holes"])
def test_rows_of_no_token_hold_nan(many_rows, holes, dev):
    """NaN in all that no token owns: tails of last pages, pages of nobody, pages whose entries are missing."""
    lengths, n, Hq, Hkv, D, page = many_rows
    c = ref.make(lengths, n, Hq, Hkv, D, page, BF16, seed=n)
    if holes:
        for s, column in ((0, 0), (0, 3), (min(1, len(lengths) - 1), 200 // page), (0, (lengths[0] - 1) // page)):
            c["table"][s, column] = -1 if column % 2 else 2 ** 31 - 1
    owned = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    for s, length in enumerate(lengths):
        for j in range(length):
            at = ref.page_of(c, s, j)
            if at is not None:
                owned[at] = True
    for t in ("k", "v"):
        c[t][~owned] = float("nan")
    out, lse = _rows(c, _to(c, dev), 40, n)
    assert out.isfinite().all() and not lse.isnan().any() and not (lse == math.inf).any()


@pytest.mark.parametrize("scale", [0.25, 0.0, -0.1])
def test_scales(many_rows, scale, dev):
    lengths, n, Hq, Hkv, D, page = many_rows
    c = ref.make(lengths, n, Hq, Hkv, D, page, BF16, seed=n + 1)
    _rows(c, _to(c, dev), 40, n, scale)


def test_infinite_and_nan_values_reach_their_own_head_only(many_rows, dev):
    """(Of one sequence they may reach rows that do not see them yet, in the same tile.)"""
    from odysseus_transformer_amd import ops
    lengths, n, Hq, Hkv, D, page = many_rows
    c = ref.make(lengths, n, Hq, Hkv, D, page, BF16, seed=n + 2)
    g = _to(c, dev)
    call = lambda: ops.paged_attn(g["q"], g["k"], g["v"], g["table"], g["lengths"])  # noqa: E731
    clean, clean_lse = call()
    G = Hq // Hkv
    g["k"][int(c["table"][0, 1]), 3, 0] = float("nan")            # place page + 3 of sequence 0: every row but the first few of a tile sees it
    g["v"][int(c["table"][0, 2]), 1, Hkv - 1] = float("inf")
    out, lse = call()
    last = slice(n - 60, n)
    assert out[0, last, :G].isnan().all() and lse[0, :G, last].isnan().all()
    if Hkv > 1:
        assert torch.equal(lse[0, G:], clean_lse[0, G:]) and torch.equal(out[0, :, G:Hq - G], clean[0, :, G:Hq - G])
        assert (out[0, last, Hq - G:] == float("inf")).all()
    assert torch.equal(out[1:], clean[1:]) and torch.equal(lse[1:], clean_lse[1:])


def test_replayed_chunks_with_other_lengths(many_rows, dev):
    """Chunks in captured graphs, two that take turns: lengths, numbers of new tokens and content are those of the replay.  Eager calls between them."""
    from odysseus_transformer_amd import ops
    lengths, n, Hq, Hkv, D, page = many_rows
    sets, graphs = [], []
    for seed in (3, 4):
        c = ref.make(lengths, n, Hq, Hkv, D, page, BF16, seed=seed)
        c["new"] = torch.tensor([n] * len(lengths), dtype=torch.int32)
        sets.append((c, _to(c, dev)))

    def step(g):
        q = ops.paged_append_(g["qkv"], Hq, g["k"], g["v"], g["table"], g["lengths"], new_tokens=g["new"])
        return ops.paged_attn(q, g["k"], g["v"], g["table"], g["lengths"], new_tokens=g["new"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _, g in sets:
            step(g)
    torch.cuda.current_stream().wait_stream(side)
    for _, g in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(g)
        graphs.append((graph, res))
    for turn in range(3):
        for (c, g), (graph, res) in zip(sets, graphs):
            now = [max(0, x - 37 * turn) for x in lengths]
            g["lengths"].copy_(torch.tensor(now, dtype=torch.int32))
            g["new"].copy_(torch.tensor([max(0, n - 29 * turn - s) for s in range(len(now))], dtype=torch.int32))
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


def test_chunks_on_two_streams_at_once(many_rows, dev):
    from odysseus_transformer_amd import ops
    lengths, n, Hq, Hkv, D, page = many_rows
    cs = [_to(ref.make(lengths, n, Hq, Hkv, D, page, BF16, seed=20 + i), dev) for i in range(2)]
    call = lambda c: ops.paged_attn(c["q"], c["k"], c["v"], c["table"], c["lengths"])  # noqa: E731
    want = [call(c) for c in cs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(cs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o, z in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(z, want[i][1])
