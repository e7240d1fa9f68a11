"""Choosing a token of each row of logits, against the definition in 64 bits on the CPU: the same tokens, and their log-probabilities."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def reference(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """tokens, logprobs in float64; and how near u is to a border between two tokens, in shares of what is kept."""
    rows, vocab = logits.shape
    of = lambda v, r, kind: kind(v[r]) if torch.is_tensor(v) else kind(v)  # noqa: E731
    tokens, logs, near = [], [], []
    for r in range(rows):
        x = logits[r].double()
        x = torch.where(torch.isnan(x), -math.inf, x) + 0.0
        single = lambda v: float(torch.tensor(float(v), dtype=F32))  # noqa: E731
        t, k, p, m = of(temperature, r, single), of(top_k, r, int), of(top_p, r, single), of(min_p, r, single)
        order = torch.sort(-x, stable=True)[1]
        x = x[order]
        if x[0] == -math.inf:
            tokens.append(-1), logs.append(-math.inf), near.append(1.0)
            continue
        if not t > 0:
            tokens.append(int(order[0])), logs.append(0.0), near.append(1.0)
            continue
        if x[0] == math.inf:
            w = (x == math.inf).double()
        else:
            d = x - x[0]
            w = torch.where(d == -math.inf, 0.0, torch.exp(d / t if math.isfinite(t) else torch.zeros_like(d)))
        n = vocab if k <= 0 else min(k, vocab)
        upto = torch.cumsum(w[:n], 0)
        before = torch.cat((torch.zeros(1, dtype=torch.float64), upto[:-1]))
        keep = torch.ones(n, dtype=torch.bool)
        if p < 1:
            keep &= before < p * upto[-1]
        if m > 0:
            keep &= w[:n] >= m
        keep[0] = True
        keep &= w[:n] > 0
        kept = torch.where(keep, w[:n], 0.0)
        upto = torch.cumsum(kept, 0)
        total = upto[-1]
        at = int((upto <= float(u[r]) * total).sum())
        at = min(at, int(keep.sum()) - 1)
        tokens.append(int(order[at])), logs.append(float(torch.log(w[at] / total)))
        near.append(float((upto / total - float(u[r])).abs()[:-1].min()) if n > 1 else 1.0)
    return torch.tensor(tokens), torch.tensor(logs, dtype=torch.float64), torch.tensor(near)


def _move(v, dev):
    return v.to(dev) if torch.is_tensor(v) else v


def check(logits, u, dev, **settings):
    """logits on the CPU, or the device's copy and what it stands for."""
    from odysseus_transformer_amd import ops
    on = logits if isinstance(logits, tuple) else (logits.to(dev), logits)
    tokens, logs = ops.sample(on[0], u.to(dev), **{k: _move(v, dev) for k, v in settings.items()})
    want, lw, _ = reference(on[1], u, **settings)
    tokens, logs = tokens.cpu(), logs.double().cpu()
    assert tokens.dtype == torch.int64 and torch.equal(tokens, want), (settings, (tokens != want).nonzero().flatten()[:8], tokens[tokens != want][:8], want[tokens != want][:8])
    # rounded once to 32 bits; the sums are of up to 2^18 weights, each off by half of 2^-44 of the largest one
    tol = 2 ** -24 * lw.abs() + 2 ** -26
    none = lw == -math.inf
    assert torch.equal(logs == -math.inf, none) and ((logs - lw).abs() <= tol)[~none].all(), (settings, (logs - lw).abs().max())


def _logits(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn((rows, vocab), generator=g)
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 12), generator=g), 9.0 * torch.rand((rows, 12), generator=g))
    return x.to(dtype), torch.rand((rows,), generator=g)


SETTINGS = [{}, dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_k=50, top_p=0.8, min_p=0.01), dict(temperature=0.0),
            dict(top_p=0.3, min_p=0.2), dict(temperature=2.0, top_k=700, top_p=0.97)]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: "_".join(f"{k}{v}" for k, v in s.items()) or "plain")
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 100), (4, 1023), (7, 1025), (3, 4099), (9, 32000), (2, 65537), (2, 131072)])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_sample(dtype, rows, vocab, settings, dev):
    logits, u = _logits(rows, vocab, dtype, seed=vocab + rows)
    check(logits, u, dev, **settings)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_each_row_has_its_own_settings(dtype, dev):
    logits, u = _logits(70, 5001, dtype, seed=1)
    g = torch.Generator().manual_seed(2)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (70,), generator=g)]  # noqa: E731
    settings = dict(temperature=pick(0.0, 0.5, 1.0, 1.7), top_k=pick(0, 1, 2, 30, 1000, 5000, 5001, 9000).to(torch.int32), top_p=pick(1.0, 0.0, 0.5, 0.99),
                    min_p=pick(0.0, 0.1, 1.0, 1e-6))
    logits[::7, 100:] = -math.inf
    check(logits, u, dev, **settings)
    for name in settings:   # numbers beside tensors
        check(logits, u, dev, **{k: v if k == name else (float if v.is_floating_point() else int)(v[3]) for k, v in settings.items()})


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1000, 9000, 40000])
def test_ties(vocab, dtype, dev):
    """Equal logits count by their index: all of them, two values, a few, steps of an eighth."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.zeros((24, vocab))
    x[8:12, ::2] = -1.0
    x[12:16] = torch.randint(0, 4, (4, vocab), generator=g).float()
    x[16:20] = torch.round(8 * torch.randn((4, vocab), generator=g)) / 8
    x[20:, vocab // 3] = 3.0
    x[4:8] = -0.0
    x[4:8, ::3] = 0.0                                     # two zeros, one value
    u = (torch.arange(24) % 8 * 2 + 1) / 16.0 + 2 ** -10
    for settings in ({}, dict(top_p=0.5), dict(top_k=vocab // 2 + 1), dict(min_p=1.0), dict(top_k=vocab // 3, top_p=0.75), dict(temperature=0.0), dict(temperature=0.1)):
        check(x.to(dtype), u, dev, **settings)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_every_token_of_a_small_vocabulary(dtype, dev):
    """Random numbers in the middle of each token's share, and right behind its border."""
    x = torch.tensor([1.0, -2.0, 0.5, 1.0, -math.inf, 0.25, 3.0, -7.0]).to(dtype)
    w = torch.exp(x.double() - 3.0)
    order = torch.sort(-x.double(), stable=True)[1]
    edges = torch.cat((torch.zeros(1, dtype=torch.float64), torch.cumsum(w[order], 0))) / w.sum()
    u = torch.cat(((edges[:-2] + edges[1:-1]) / 2, edges[:-2] + 2 ** -22, torch.tensor([0.0, 1 - 2 ** -24, 1.0]).double())).float()
    check(x.expand(len(u), -1).contiguous(), u, dev)
    tokens, _, _ = reference(x.expand(7, -1), u[:7])
    assert torch.equal(tokens, order[:7])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_masked_infinite_and_nan_logits(dtype, dev):
    logits, u = _logits(12, 3000, dtype, seed=4)
    lowest = torch.finfo(dtype).min
    logits[0] = -math.inf                                   # nothing left
    logits[1] = math.nan
    logits[2, :] = -math.inf
    logits[2, 2999] = -5.0                                  # one left
    logits[3, 7] = math.inf
    logits[4, ::100] = math.inf                             # several share all of it
    logits[5, ::2] = math.nan
    logits[6, 10:] = lowest
    logits[7] = lowest
    logits[8, 5:] = -math.inf                               # fewer than top_k
    logits[9, :2500] = lowest
    logits[10, ::3] = -1e30
    for settings in SETTINGS:
        check(logits, u, dev, **settings)
    check(logits, torch.zeros(12), dev, top_k=20, top_p=0.5)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 30.0, 1e4, 1e30, math.inf])
def test_temperatures_far_from_one(temperature, dtype, dev):
    """Nothing but the largest, and buckets of too many tokens to be sorted: they are divided by the bits of the values."""
    logits, u = _logits(6, 20000, dtype, seed=7)
    for settings in ({}, dict(top_k=3), dict(top_k=9000), dict(top_p=0.4), dict(min_p=0.999), dict(top_k=15000, top_p=0.9, min_p=1e-3)):
        check(logits, u, dev, temperature=temperature, **settings)


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 300.0, 1e30])
def test_logits_of_other_sizes(scale, dev):
    logits, u = _logits(5, 30000, F32, seed=8)
    for settings in ({}, dict(top_k=50), dict(top_k=12000, top_p=0.7), dict(top_p=0.6), dict(min_p=0.3)):
        check(logits * scale + 5.0, u, dev, **settings)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_rows_that_are_not_aligned(dtype, dev):
    """The last token's logits of a padded batch, slices, odd strides: what lies around a row is not looked at."""
    from odysseus_transformer_amd import ops
    wide = torch.full((4, 3, 1111), math.inf).to(dtype)
    small, u = _logits(4, 1001, dtype, seed=9)
    on = wide.to(dev)
    for first in range(9):
        on.fill_(math.inf)
        view = on[:, -1, first:first + 1001]
        view.copy_(small)
        check((view, small), u, dev, top_k=30, top_p=0.9)
        check((view, small), u, dev)
    flat = torch.full((5000,), math.nan, device=dev, dtype=dtype)
    for first in (0, 1, 5):
        flat[first:first + 1001] = small[0]
        check((flat[first:first + 1001][None], small[:1]), u[:1], dev)
    lone = torch.zeros((1, 1), dtype=dtype, device=dev)
    assert ops.sample(lone, u[:1].to(dev))[0].item() == 0


def test_largest_vocabularies(dev):
    for vocab in (262144, 2 ** 21 - 4):
        for dtype in (BF16, F32):
            logits, u = _logits(1, vocab, dtype, seed=3)
            for settings in ({}, dict(top_k=50), dict(top_p=0.95), dict(temperature=50.0, top_k=100000)):
                check(logits, u, dev, **settings)
            check(torch.zeros_like(logits), u, dev)


def test_equal_in_any_batch_and_again(dev):
    """A row's result does not go by its batch, and a call gives the same twice: sums are of whole numbers."""
    from odysseus_transformer_amd import ops
    logits, u = _logits(300, 33000, BF16, seed=5)
    logits, u = logits.to(dev), u.to(dev)
    for settings in ({}, dict(top_p=0.9), dict(top_k=100, min_p=0.001)):
        whole = ops.sample(logits, u, **settings)
        again = ops.sample(logits, u, **settings)
        assert torch.equal(whole[0], again[0]) and torch.equal(whole[1], again[1])
        for r in (0, 17, 299):
            lone = ops.sample(logits[r:r + 1], u[r:r + 1], **settings)
            assert torch.equal(lone[0], whole[0][r:r + 1]) and torch.equal(lone[1], whole[1][r:r + 1])


def test_shares_of_many_draws(dev):
    """What each token is drawn, of evenly spread random numbers: its share to one in their number."""
    from odysseus_transformer_amd import ops
    logits, _ = _logits(1, 50, F32, seed=6)
    n = 20000
    u = (torch.arange(n) + 0.5) / n
    tokens, _ = ops.sample(logits.to(dev).expand(n, -1).contiguous(), u.to(dev), temperature=0.8)
    share = torch.bincount(tokens.cpu(), minlength=50).double() / n
    assert ((share - torch.softmax(logits[0].double() / float(torch.tensor(0.8)), 0)).abs() <= 1.01 / n).all()


def test_both_host_paths_agree(dev, monkeypatch):
    from odysseus_transformer_amd import _native, ops
    logits, u = _logits(5, 1000, BF16, seed=1)
    logits, u = logits.to(dev), u.to(dev)
    t = torch.full((5,), 0.7, device=dev)
    k = torch.full((5,), 30, device=dev, dtype=torch.int32)
    calls = [dict(), dict(temperature=t, top_k=k), dict(temperature=0.7, top_k=30, top_p=t, min_p=0), dict(temperature=1, top_p=1)]
    plain = [ops.sample(logits, u, **c) for c in calls]
    monkeypatch.setattr(ops, "native", _native._Nothing())
    for c, (a, b) in zip(calls, plain):
        x, y = ops.sample(logits, u, **c)
        assert torch.equal(a, x) and torch.equal(b, y)


def test_replayed_from_a_graph(dev):
    from odysseus_transformer_amd import ops
    logits, u = _logits(9, 20000, BF16, seed=2)
    x, v = logits.to(dev), u.to(dev)
    p = torch.full((9,), 0.9, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample(x, v, top_p=p)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.sample(x, v, top_p=p), ops.sample(x, v, top_k=20)
    for turn in range(3):
        x.copy_(_logits(9, 20000, BF16, seed=20 + turn)[0])
        v.copy_(torch.rand(9))
        p.fill_(0.9 - 0.2 * turn)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, (ops.sample(x, v, top_p=p), ops.sample(x, v, top_k=20))):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_calls_on_two_streams_at_once(dev):
    from odysseus_transformer_amd import ops
    sets = [tuple(t.to(dev) for t in _logits(40, 32000, BF16, seed=i)) for i in range(2)]
    want = [ops.sample(*s, top_p=0.9) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(4):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(ops.sample(*s, top_p=0.9))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 2][0]) and torch.equal(b, want[i % 2][1])


def test_nothing_to_do_and_refusals(dev):
    from odysseus_transformer_amd import _lib, ops
    logits, u = _logits(4, 100, BF16, seed=1)
    x, v = logits.to(dev), u.to(dev)
    tokens, logs = ops.sample(x[:0], v[:0])
    assert tokens.shape == logs.shape == (0,)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0), dict(temperature=math.nan), dict(top_k=2 ** 31),
                dict(temperature=torch.ones(3, device=dev)), dict(temperature=torch.ones(4, device=dev).double()), dict(top_k=torch.ones(4, device=dev)),
                dict(top_p=torch.ones(8, device=dev)[::2])):
        with pytest.raises(ValueError):
            ops.sample(x, v, **bad)
    for bad in (lambda: ops.sample(x, v[:3]), lambda: ops.sample(x, v.double()), lambda: ops.sample(x[0], v), lambda: ops.sample(x[:, :0], v), lambda: ops.sample(x.t(), v),
                lambda: ops.sample(x[:1].expand(4, -1), v)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.sample(x, u)
    with pytest.raises(RuntimeError):
        ops.sample(x, v, top_p=torch.ones(4))
    with pytest.raises(TypeError):
        ops.sample(x.half(), v)
    with pytest.raises(TypeError):
        ops.sample(x, 0.5)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.sample(x.clone().requires_grad_(), v)
    with torch.no_grad():
        ops.sample(x.clone().requires_grad_(), v)
    with pytest.raises(_lib.OdysseusHipError, match="rows of"):
        ops.sample(torch.empty((1, 2 ** 21), dtype=BF16, device=dev), v[:1])


# ------------------------------------------------------------------------------------------------ few long rows, which are divided among blocks
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [65536, 98304, 131077])
def test_long_rows_of_all_kinds(vocab, dtype, dev):
    """Rows side by side that are divided differently: greedy, few of top_k, more, none; of -inf, with +inf, NaN, equals, what one slice alone has."""
    rows = 30
    logits, u = _logits(rows, vocab, dtype, seed=vocab)
    g = torch.Generator().manual_seed(3)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)]  # noqa: E731
    settings = dict(temperature=pick(0.0, 0.6, 1.0, 1.7), top_k=pick(0, 0, 1, 40, 2048, 2049, vocab - 1).to(torch.int32), top_p=pick(1.0, 0.5, 0.95), min_p=pick(0.0, 0.0, 0.02))
    logits[1] = -math.inf
    logits[2, ::vocab // 7] = math.inf
    logits[3, ::3] = math.nan
    logits[4] = 1.25
    logits[5, vocab // 2:] = -math.inf
    logits[6, :vocab - 5] = -math.inf
    logits[7] = torch.round(logits[7])
    logits[8] = 3.0
    logits[8, vocab - 1] = 4.0
    logits[9] *= 60.0
    logits[10] *= 1e-3
    logits[11, 100:] = -math.inf
    logits[13], logits[14] = 0.0, -0.0
    logits[14, ::5] = -1.0
    logits[15] = -logits[15].abs() - 1.0
    logits[16, ::2] *= 1e-9
    logits[12, 1:] = -3e38 if dtype == F32 else -300.0
    check(logits, u, dev, **settings)
    for name in settings:
        check(logits, u, dev, **{name: settings[name]})
    check(logits, u, dev)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_long_rows_are_equal_in_any_batch(dtype, dev):
    from odysseus_transformer_amd import ops
    logits, u = _logits(300, 100003, dtype, seed=5)
    logits, u = logits.to(dev), u.to(dev)
    for settings in ({}, dict(top_p=0.9), dict(top_k=100, min_p=0.001), dict(temperature=0.0), dict(min_p=0.01, top_p=0.99)):
        whole = ops.sample(logits, u, **settings)
        for part in (slice(0, 1), slice(17, 40), slice(100, 220)):
            some = ops.sample(logits[part], u[part], **settings)
            assert torch.equal(some[0], whole[0][part]) and torch.equal(some[1], whole[1][part])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_long_rows_that_are_not_aligned(dtype, dev):
    logits, u = _logits(5, 98333, dtype, seed=9)
    for shift in (1, 2, 3, 5):
        wide = torch.full((5, 98333 + 8), math.inf, dtype=dtype)
        wide[:, shift:shift + 98333] = logits
        on = wide.to(dev)[:, shift:shift + 98333]
        check((on, logits), u, dev, top_p=0.9)
        check((on, logits), u, dev, top_k=30)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_long_rows_replayed_and_on_two_streams(dtype, dev):
    from odysseus_transformer_amd import ops
    sets = [tuple(t.to(dev) for t in _logits(4, 100001, dtype, seed=i)) for i in range(2)]
    calls = [dict(top_p=0.9), dict(top_k=20), dict()]
    want = [[ops.sample(*s, **c) for c in calls] for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(4):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append([ops.sample(*s, **c) for c in calls])
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        for (a, b), (c, d) in zip(results, want[i % 2]):
            assert torch.equal(a, c) and torch.equal(b, d)
    x, v = (t.clone() for t in sets[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [ops.sample(x, v, **c) for c in calls]
    for turn in range(4):
        x.copy_(sets[turn % 2][0])
        v.copy_(sets[turn % 2][1])
        graph.replay()
        torch.cuda.synchronize()
        eager = [ops.sample(x, v, **c) for c in calls]
        for (a, b), (c, d), (e, f) in zip(captured, want[turn % 2], eager):
            assert torch.equal(a, c) and torch.equal(b, d) and torch.equal(e, c) and torch.equal(f, d)


def test_long_rows_by_both_host_paths(dev, monkeypatch):
    from odysseus_transformer_amd import _native, ops
    for dtype in (BF16, F32):
        logits, u = (t.to(dev) for t in _logits(3, 100001, dtype, seed=4))
        plain = [ops.sample(logits, u, **c) for c in (dict(top_p=0.9), dict(top_k=30))]
        with monkeypatch.context() as m:
            m.setattr(ops, "native", _native._Nothing())
            for c, (a, b) in zip((dict(top_p=0.9), dict(top_k=30)), plain):
                x, y = ops.sample(logits, u, **c)
                assert torch.equal(a, x) and torch.equal(b, y)
