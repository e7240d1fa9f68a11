"""PagedKVCache in 8 bits: its book-keeping, and what the entry points refuse before anything reaches a device (CPU); layers over it, and a decoding loop that
chooses its next tokens (GPU)."""
import math
import re

import pytest
import torch

from odysseus_transformer_amd.utils.paged_cache import PagedKVCache
from test_product_distances import _assembly, _kernels, M0, test_wait_states_around_products_by_hand as _wait_states

BF16, F32, F8, E8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _book(**kw):
    args = dict(num_layers=2, num_pages=10, max_sequences=3, max_length=100, n_kv_heads=2, head_dim=64, page_size=16, device="cpu", dtype=F8)
    return PagedKVCache(**{**args, **kw})


def test_pools_and_scales():
    c = _book()
    (k, v), (kz, vz) = c.layer(1), c.scales(1)
    assert c.in_8_bits and c.scale_block == 16 and k.dtype == v.dtype == F8 and kz.dtype == vz.dtype == E8
    assert k.shape == (10, 16, 2, 64) and kz.shape == vz.shape == (10, 1, 2) and kz.data_ptr() != c.scales(0)[0].data_ptr()
    c = _book(page_size=64, scale_block=8)
    assert c.scales(0)[0].shape == (10, 8, 2) and _book(page_size=128).scale_block == 32
    c.begin([33, 5])
    assert c.lengths.tolist() == [33, 5, 0]
    for bad in (dict(scale_block=4), dict(scale_block=32), dict(scale_block=24, page_size=64), dict(scale_block=128, page_size=256), dict(scale_block=16, dtype=BF16)):
        with pytest.raises(ValueError):
            _book(**bad)
    plain = _book(dtype=BF16)
    assert not plain.in_8_bits
    for call in (lambda: plain.scales(0), lambda: plain.values(0)):
        with pytest.raises(ValueError):
            call()


def test_entry_points_refuse_without_a_gpu():
    from odysseus_transformer_amd import ops
    c = _book()
    c.begin([4, 4, 4])
    where = (*c.layer(0), *c.scales(0), c.page_table, c.lengths)
    for call in (lambda: ops.paged_append_q8_(torch.zeros(3, 1, 6, 64, dtype=BF16), 2, *where), lambda: ops.paged_attn_q8(torch.zeros(3, 1, 2, 64, dtype=BF16), *where),
                 lambda: ops.paged_read_q8(*where, 4), lambda: c.values(0), lambda: ops.sample(torch.zeros(2, 5), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


Q = 16            # an aligned address that nothing is read from


def _code(name, S=1, n=1, Hq=4, Hkv=2, D=64, pages=4, page=16, block=8, width=3, dtype=0, scales=Q, misaligned=True):
    """The status of a call whose pages are misaligned (-3, the last of the checks that all share), or, if not, of one that a later check refuses."""
    from odysseus_transformer_amd import _lib
    xs, ps, zs = (512, 512, 64), (1 << 20, 130 if misaligned else 128, 64), (16, 2, 1)
    with pytest.raises(_lib.OdysseusHipError) as e:
        if name == "ody_paged_append_q8":
            _lib.call(name, Q, Q, Q, Q, scales, Q, Q, Q, 0, 0, 0, S, n, Hq, Hkv, D, *xs, *xs, *ps, *ps, *zs, *zs, pages, page, block, width, width, dtype, 0)
        elif name == "ody_paged_read_q8":
            _lib.call(name, Q, Q, scales, Q, Q, Q, 0, 0, S, 5, Hkv, D, *ps, *ps, *zs, *zs, pages, page, block, width, width, dtype, 0)
        else:
            _lib.call(name, 0, Q, Q, scales, Q, Q, Q, 0, Q, Q, S, n, Hq, Hkv, D, *xs, *ps, *ps, *zs, *zs, *xs, pages, page, block, width, width, 1.0, dtype, 0, 0, 0)
    return e.value.code


@pytest.mark.parametrize("name", ["ody_paged_append_q8", "ody_paged_read_q8", "ody_paged_attn_q8"])
def test_refusals_of_the_entry_points(name):
    assert _code(name) == -3
    assert _code(name, misaligned=False) == -4                     # what comes next is NULL
    for sizes, code in ((dict(S=0), -1), (dict(pages=0), -1), (dict(width=0), -1), (dict(Hkv=0), -1), (dict(D=96), -2), (dict(dtype=2), -2), (dict(page=12), -2), (dict(page=4), -2),
                        (dict(width=2 ** 27), -1)):
        assert _code(name, **sizes) == code, sizes
    for sizes, code in ((dict(block=4), -2), (dict(block=12), -2), (dict(block=32), -2), (dict(block=128, page=256), -2), (dict(scales=0), -4)):
        assert _code(name, misaligned=False, **sizes) == code, sizes
    most = (2 ** 31 - 4096) // 16
    assert _code(name, width=most) == -3 and _code(name, width=most + 1) == -1


def test_tokens_of_one_launch():
    from odysseus_transformer_amd import _lib
    for S, n, block, code in ((1 << 14, 1 << 10, 8, -1), (1 << 23, 1, 8, -1), (1 << 22, 2, 8, -1), ((1 << 23) - 1, 1, 8, -4), (1 << 12, (1 << 12) - 1, 16, -4)):
        with pytest.raises(_lib.OdysseusHipError) as e:   # -4: there is no projection
            _lib.call("ody_paged_append_q8", 0, Q, Q, Q, Q, Q, Q, Q, 0, 0, Q, S, n, 2, 1, 64, *(256, 256, 64) * 2, *(2048, 64, 64) * 2, *(2, 1, 1) * 2, 4, 16, block, 3, 3, 0, 0)
        assert e.value.code == code, (S, n)


def test_refusals_of_sampling():
    from odysseus_transformer_amd import _lib

    def code(logits=Q, u=Q, tokens=Q, rows=1, vocab=10, stride=10, dtype=0, workspace=0, space=0):
        with pytest.raises(_lib.OdysseusHipError) as e:
            _lib.call("ody_sample", logits, u, 0, 0, 0, 0, 1.0, 0, 1.0, 0.0, tokens, Q, rows, vocab, stride, dtype, workspace, space, 0)
        return e.value.code
    assert code(logits=0) == code(u=0) == code(tokens=0) == -4
    assert code(rows=0) == code(vocab=0) == code(vocab=2 ** 21 - 3) == code(rows=1 << 22) == code(rows=2, stride=9) == -1
    assert code(dtype=3) == -2
    assert code(logits=17) == code(logits=18, dtype=1) == -3
    need = _lib.load().ody_sample_workspace_bytes(2, 100000, 1)
    assert need > 0 and _lib.load().ody_sample_workspace_bytes(2, 1000, 1) == _lib.load().ody_sample_workspace_bytes(0, 100000, 1) == 0
    for bad in (dict(), dict(workspace=4096, space=need - 1), dict(workspace=4096 + 128, space=need), dict(space=need)):
        assert code(rows=2, vocab=100000, stride=100000, dtype=1, **bad) == -5, bad


def test_m0_belongs_to_the_direct_loads(tmp_path):
    """As in the kernels over a cache in 16 bits: a value that the compiler kept in m0 would be lost."""
    loads = 0
    for name, code, _ in _kernels(_assembly("paged_q8_chunk", tmp_path)):
        for op, operands, by_hand in code:
            if by_hand:
                loads += op.startswith("global_load_lds")
            else:
                assert not M0.match(op) and not any(re.search(r"\bm0\b|\blds$", o) for o in operands), f"{name}: {op} {operands}"
    assert loads >= 20


def test_wait_states_around_products(tmp_path):
    _wait_states("paged_q8_wide", tmp_path)


# ------------------------------------------------------------------------------------------------ on the GPU
def _cache(dtype_, D, dev, **kw):
    args = dict(num_layers=1, num_pages=40, page_size=16, max_sequences=3, max_length=200, n_kv_heads=2, head_dim=D, dtype=F8, device=dev, scale_block=8)
    return PagedKVCache(**{**args, **kw})


def _attention_over(cache, layer, x, s):
    """The attention module's result for a sequence's tokens x (n, hidden), in float64 on the CPU, over what the cache holds of it, themselves included."""
    from odysseus_transformer_amd import ops
    a = layer.self_attn
    nh, nkv, D = a.num_heads, a.num_key_value_heads, a.head_dim
    k, v = (t[s].double().cpu() for t in cache.values(0, F32))
    length, n = cache.sequence_lengths()[s], x.shape[0]
    q = (x.double() @ a.qkv_proj.weight.double().cpu()[:nh * D].t()).view(n, nh, D)
    at = torch.arange(length - n, length)
    th = torch.outer(at.double(), 1.0 / (10000.0 ** (torch.arange(0, D, 2).double() / D)))
    cos, sin = torch.cat((th.cos(), th.cos()), -1)[:, None], torch.cat((th.sin(), th.sin()), -1)[:, None]
    q = q * cos + torch.cat((-q[..., D // 2:], q[..., :D // 2]), -1) * sin
    out = torch.empty(n, nh, D, dtype=torch.float64)
    for i in range(n):
        for h in range(nh):
            e = length - n + i + 1
            p = torch.softmax(k[:e, h * nkv // nh] @ q[i, h] / math.sqrt(D), 0)
            out[i, h] = p @ v[:e, h * nkv // nh]
    return out.reshape(n, nh * D) @ a.o_proj.weight.double().cpu().t()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (F32, 64)], ids=["bf16_128", "bf16_64", "f32"])
def test_attention_module_over_a_cache_in_8_bits(dtype, D, dev):
    """Prompts of different lengths, single tokens, a few at once, tokens that are taken back, a sequence in another's place: every result is the formula's over
    the values that the cache holds; and those are the projection's, to half a step of eight bits."""
    from test_paged_gpu import _layer, _tol
    layer, cache = _layer(dtype, D, dev), _cache(dtype, D, dev)
    g = torch.Generator().manual_seed(5)
    largest = 0.0                                                   # of the values so far
    for new in ([70, 9, 33], [1, 1, 1], [1, 0, 1], [0, 20, 1], [66, 5, 2], "truncate", [40, 1, 1], "free", [1, 50, 0], [1, 1, 1]):
        if new == "truncate":
            cache.truncate(0, cache.sequence_lengths()[0] - 40)
            continue
        if new == "free":
            cache.free(1)
            continue
        n, fresh = cache.begin(new), cache.fresh
        x = torch.randn(3, n, 256, generator=g).to(dtype)
        with torch.no_grad():
            y = layer.self_attn(x.to(dev), past_key_value=cache)[0].double().cpu()
        assert y.isfinite().all()
        v = (x.double() @ layer.self_attn.qkv_proj.weight.double().cpu()[-2 * D:].t()).view(3, n, 2, D)
        largest = max(largest, v.abs().max().item())
        for s, t in enumerate(new):
            if t:
                if not fresh:                                       # (a prompt of a new sequence reads the tokens at hand)
                    want = _attention_over(cache, layer, x[s, n - t:], s)
                    assert (y[s, n - t:] - want).norm() <= _tol(dtype) * want.norm(), f"step {new}, sequence {s}"
                mine, length = v[s, n - t:], cache.sequence_lengths()[s]
                held = cache.values(0, F32)[1][s, length - t:length].double().cpu()
                # half a step of eight bits: 2^-4 of a value, or 2^-10 of a scale below largest / 224, and as much again where a later token raises the scale;
                # the projection's own rounding to 16 bits, 2^-8, and its sums in 32
                assert ((held - mine).abs() <= (2 ** -4 + 2 ** -7) * mine.abs() + 2 ** -9 * largest / 224 + 2 ** -16 * mine.norm(dim=-1, keepdim=True)).all()


@pytest.mark.gpu
def test_decoder_layer_takes_it_as_the_other_cache(dev):
    """A whole layer's rows next to those over a cache in 16 bits: as near as eight bits of keys and values let them be."""
    from test_paged_gpu import _cache as plain_cache, _layer
    layer = _layer(BF16, 128, dev)
    a, b = _cache(BF16, 128, dev), plain_cache(BF16, 128, dev)
    x = torch.randn(3, 60, 256, generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    for new in ([30, 30, 30], [20, 3, 7], 1, 1):
        n = [c.begin(new) for c in (a, b)][0]
        with torch.no_grad():
            ya, yb = layer(x[:, :n], past_key_values=a), layer(x[:, :n], past_key_values=b)
        if new == [30, 30, 30]:
            assert torch.equal(ya, yb)   # a fresh prompt reads the tokens at hand
        else:
            # a step of 2^-4 of a value at most, half of it on average less, in keys and in values, of a residual stream that is larger than either
            assert (ya.float() - yb.float()).norm() <= 0.08 * yb.float().norm()


@pytest.mark.gpu
def test_captured_step_is_replayed_behind_begin(dev):
    from test_paged_gpu import _layer
    layer = _layer(BF16, 128, dev)
    caches = [_cache(BF16, 128, dev) for _ in range(2)]
    x = torch.randn(3, 60, 256, generator=torch.Generator().manual_seed(8)).to(BF16).to(dev)
    for c in caches:
        n = c.begin([20, 3, 31])
        with torch.no_grad():
            layer(x[:, :n], past_key_values=c)
    static = torch.zeros(3, 1, 256, dtype=BF16, device=dev)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    caches[0].begin(1)
    with torch.no_grad():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(static, past_key_values=caches[0])   # of zeros: leaves no scale larger than what follows needs
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            y = layer(static, past_key_values=caches[0])
    for s, length in enumerate((20, 3, 31)):
        caches[0].truncate(s, length)
    for t in range(5):
        new = [1, 1, 1] if t != 3 else [1, 0, 1]
        static.copy_(x[:, 40 + t:41 + t])
        caches[0].begin(new)
        graph.replay()
        caches[1].begin(new)
        with torch.no_grad():
            z = layer(x[:, 40 + t:41 + t], past_key_values=caches[1])
        for s in range(3):
            if new[s]:
                assert torch.equal(y[s], z[s]), (t, s)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            caches[0].values(0)


@pytest.mark.gpu
def test_decoding_loop(dev):
    """What a program runs: prompts, then steps of append, attention and a head's logits, of which the next tokens are sampled -- eager, and with the step captured:
    the same tokens; and each is the definition's for its logits."""
    from odysseus_transformer_amd import ops
    from test_paged_gpu import _layer
    from test_sample_gpu import reference
    layer, vocab, S = _layer(BF16, 128, dev), 1000, 3
    g = torch.Generator().manual_seed(11)
    embed = torch.randn(vocab, 256, generator=g).to(BF16).to(dev)
    head = (0.3 * torch.randn(vocab, 256, generator=g)).to(BF16).to(dev)
    prompt = torch.randint(0, vocab, (S, 25), generator=g).to(dev)
    u = torch.rand(12, S, generator=g).to(dev)
    settings = dict(temperature=torch.tensor([0.7, 1.0, 0.0], device=dev), top_k=torch.tensor([0, 50, 0], dtype=torch.int32, device=dev), top_p=0.9, min_p=0.01)

    def step(tokens, cache, draw):
        y = layer(embed[tokens], past_key_values=cache)
        logits = ops.gemm(0, y[:, -1], head)                # the last token's
        return (logits, *ops.sample(logits, draw, **settings))

    def run(captured):
        cache, said = _cache(BF16, 128, dev), []
        cache.begin([25, 7, 16])
        logits, tokens, logs = step(prompt, cache, u[0])
        graph = None
        for t in range(1, 12):
            said.append((logits.clone(), tokens.clone(), logs.clone()))
            cache.begin(1)
            if not captured:
                logits, tokens, logs = step(tokens[:, None], cache, u[t])
                continue
            if graph is None:
                ids, draw = tokens[:, None].clone(), u[t].clone()
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step(ids, cache, draw)
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    logits, tokens, logs = step(ids, cache, draw)
            ids.copy_(said[-1][1][:, None])
            draw.copy_(u[t])
            graph.replay()
        said.append((logits.clone(), tokens.clone(), logs.clone()))
        return said
    with torch.no_grad():
        eager, replayed = run(False), run(True)
    for t, ((logits, tokens, logs), (_, again, logs_again)) in enumerate(zip(eager, replayed)):
        want = reference(logits.cpu(), u[t].cpu(), **{k: v.cpu() if torch.is_tensor(v) else v for k, v in settings.items()})[0]
        assert torch.equal(tokens.cpu(), want) and torch.equal(tokens, again) and torch.equal(logs, logs_again), t
