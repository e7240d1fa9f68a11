"""The host side of a key / value cache in pages: its book-keeping, and what the entry points refuse before anything reaches a device."""
import types

import pytest
import torch

from odysseus_transformer_amd.utils.paged_cache import PagedKVCache


def _cache(**kw):
    args = dict(num_layers=2, num_pages=10, max_sequences=3, max_length=100, n_kv_heads=2, head_dim=64, page_size=16, device="cpu")
    return PagedKVCache(**{**args, **kw})


def _check(cache):
    """Every page belongs to one sequence or to nobody; the table says what the book says."""
    owned = [p for pages in cache._owned for p in pages]
    assert sorted(owned + cache._free) == list(range(cache.num_pages))
    for s, pages in enumerate(cache._owned):
        row = cache.page_table[s].tolist()
        assert row[:len(pages)] == pages and all(p == -1 for p in row[len(pages):])
        assert len(pages) == -(-cache._length[s] // cache.page_size)


def test_steps():
    c = _cache()
    k, v = c.layer(1)
    assert k.shape == v.shape == (10, 16, 2, 64) and k.data_ptr() != c.layer(0)[0].data_ptr()
    assert c.begin([33, 5]) == 33
    _check(c)
    assert c.lengths.tolist() == [33, 5, 0] and c.new_tokens.tolist() == [33, 5, 0] and not c.fresh
    assert c.sequence_lengths() == [33, 5, 0] and c.get_seq_length() == 0
    assert c.position_ids.shape == (3, 33) and c.position_ids[0].tolist() == list(range(33)) and c.position_ids[1, 28:].tolist() == list(range(5))
    held = c.page_table, c.lengths, c.new_tokens
    at = c.position_ids.data_ptr()
    assert c.begin(1) == 1                                   # only sequences that have begun
    assert c.lengths.tolist() == [34, 6, 0] and c.new_tokens.tolist() == [1, 1, 0] and c.position_ids[:, 0].tolist() == [33, 5, 0]
    assert c.get_seq_length() == 33
    c.begin([0, 7, 2])                                       # one stands still, one goes on, one begins
    assert c.lengths.tolist() == [0, 13, 2] and c.new_tokens.tolist() == [0, 7, 2] and c.sequence_lengths() == [34, 13, 2]
    assert c.position_ids[1].tolist() == list(range(6, 13))
    c.begin([33])
    assert c.page_table is held[0] and c.lengths is held[1] and c.new_tokens is held[2] and c.position_ids.data_ptr() == at   # a captured step reads them again
    _check(c)
    c.free(0)
    _check(c)
    assert c.lengths.tolist() == [0, 0, 0] and c.sequence_lengths() == [0, 13, 2]
    c.truncate(1, 6)
    c.begin(torch.tensor([4, 1, 1]))
    assert c.lengths.tolist() == [4, 7, 3]
    _check(c)


def test_fresh_steps():
    c = _cache()
    c.begin([20, 20, 20])
    assert c.fresh
    c.begin(1)
    assert not c.fresh
    c.begin([0, 0, 0, ][:2] + [1])
    assert not c.fresh
    for s in range(3):
        c.free(s)
    c.begin([20, 20])                                        # the third row takes no part
    assert not c.fresh


def test_refused_steps_change_nothing():
    c = _cache()
    c.begin([90, 30])                                        # 6 + 2 pages of 10
    before = c.page_table.clone(), c.lengths.clone(), c.sequence_lengths(), c.free_pages()
    for bad, error in (([11], ValueError), ([1, 1, 33], MemoryError), ([1, 2, 3, 4], ValueError), ([-1, 2], ValueError), ([0, 0], ValueError), (0, ValueError)):
        with pytest.raises(error):
            c.begin(bad)
        assert torch.equal(c.page_table, before[0]) and torch.equal(c.lengths, before[1])
        assert c.sequence_lengths() == before[2] and c.free_pages() == before[3]
    _check(c)
    for s, length in ((3, 0), (-1, 0), (0, 91), (0, -1)):
        with pytest.raises(ValueError):
            c.truncate(s, length)
    with pytest.raises(ValueError):
        _cache().begin(1)                                    # nothing has begun
    for kw in (dict(page_size=12), dict(page_size=4), dict(num_pages=0), dict(max_sequences=0), dict(head_dim=-1)):
        with pytest.raises(ValueError):
            _cache(**kw)


def _module():
    from odysseus_transformer_amd.decoder.odysseus import LlamaFlashAttention2TPSP
    cfg = types.SimpleNamespace(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=256, hidden_act="silu",
                                attention_dropout=0.1, rms_norm_eps=1e-6, rope_theta=10000.0, pretraining_tp=1)
    return LlamaFlashAttention2TPSP(cfg, 1)


def test_module_refusals():
    m, c = _module(), _cache(dtype=torch.float32)
    x = torch.zeros(3, 5, 128)
    with pytest.raises(ValueError, match="eval"):            # training with dropout
        m(x, past_key_value=c)
    m.eval()
    with pytest.raises(ValueError, match="begin"):
        m(x, past_key_value=c)
    c.begin([5, 5, 5])
    with pytest.raises(ValueError, match="begin"):
        m(x[:2], past_key_value=c)
    with pytest.raises(ValueError, match="attention_mask"):
        m(x, past_key_values=c, attention_mask=torch.ones(3, 5))
    with pytest.raises(RuntimeError, match="HIP device"), torch.no_grad():
        m(x, past_key_values=c)


def test_entry_points_refuse_without_a_gpu():
    from odysseus_transformer_amd import _lib, ops
    A, Q, D = _lib.load(), 16, 64                            # an aligned address that nothing is read from
    shape = dict(S=2, n=1, Hq=4, Hkv=2, D=64, pages=4, page=16, width=3, tstride=3, dtype=0, xs=(512, 512, 64), ps=(2048, 128, 64), scale=1.0)

    def append(k=Q, q=Q, x=Q, f=Q, **kw):
        a = {**shape, **kw}
        _lib.call("ody_paged_append", x, q, k, Q, Q, Q, 0, 0, f, a["S"], a["n"], a["Hq"], a["Hkv"], a["D"], *a["xs"], *a["xs"], *a["ps"], *a["ps"], a["pages"],
                  a["page"], a["width"], a["tstride"], a["dtype"], 0)

    def attn(k=Q, q=Q, x=Q, f=Q, ws=0, ws_bytes=0, **kw):
        a = {**shape, **kw}
        _lib.call("ody_paged_attn", x, k, Q, Q, Q, 0, q, f, a["S"], a["n"], a["Hq"], a["Hkv"], a["D"], *a["xs"], *a["ps"], *a["ps"], *a["xs"], a["pages"], a["page"],
                  a["width"], a["tstride"], a["scale"], a["dtype"], ws, ws_bytes, 0)

    bad = [(dict(k=0), -4), (dict(x=0), -4), (dict(f=0), -4), (dict(S=0), -1), (dict(n=-1), -1), (dict(pages=0), -1), (dict(width=0), -1), (dict(Hkv=3), -1),
           (dict(D=96), -2), (dict(dtype=2), -2), (dict(page=12), -2), (dict(page=4), -2), (dict(page=0), -2), (dict(tstride=2), -1),
           (dict(width=1 << 28, tstride=1 << 28), -1), (dict(S=1 << 20, n=1 << 10), -1), (dict(xs=(512, 512, 60)), -3), (dict(ps=(2048, 130, 64)), -3),
           (dict(k=24), -3), (dict(ps=(1 << 31, 128, 64)), -2), (dict(ps=(2048, 1 << 28, 64)), -2)]
    for call in (append, attn):
        for kw, code in bad:
            with pytest.raises(_lib.OdysseusHipError) as e:
                call(**kw)
            assert e.value.code == code, (call.__name__, kw, e.value.msg)
    need = A.ody_paged_attn_workspace_bytes(2, 1, 4, 2, 64, 16, 64, 0)
    assert need > 0 and A.ody_paged_attn_workspace_bytes(2, 1, 4, 2, 64, 16, 8, 0) == 0   # 128 keys are one step: nothing to be joined
    for ws, n in ((0, 0), (256, need - 1), (128, need)):
        with pytest.raises(_lib.OdysseusHipError) as e:
            attn(width=64, tstride=64, ws=ws, ws_bytes=n)
        assert e.value.code == -5
    with pytest.raises(_lib.OdysseusHipError) as e:          # more steps than can be counted
        attn(S=1 << 22, width=1 << 20, tstride=1 << 20)
    assert e.value.code == -1
    x = torch.zeros(2, 1, 8, 64)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.paged_append_(x, 4, x, x, x, x)
    with pytest.raises(ValueError, match="rotation"):
        ops.paged_append_(x, 4, x, x, x, x, position_ids=torch.zeros(2, 1), rotate=False)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.paged_attn(x, x, x, x, x)


def test_a_layer_without_an_index_over_a_cache_of_several():
    """Modules that do not say which layer they are would share one layer's pages, and overwrite each other's keys."""
    m, c = _module().eval(), _cache(dtype=torch.float32)
    c.begin([5, 5, 5])
    x = torch.zeros(3, 5, 128)
    m.layer_idx = None
    with pytest.raises(ValueError, match="layer_idx"), torch.no_grad():
        m(x, past_key_values=c)
    one = _cache(dtype=torch.float32, num_layers=1)
    one.begin([5, 5, 5])
    m.layer_idx = None
    with pytest.raises(RuntimeError, match="HIP device"), torch.no_grad():   # a lone layer needs none
        m(x, past_key_values=one)


def test_no_step_behind_truncate():
    """A sequence whose new tokens were taken back has none: a step that runs before the next begin() would leave it out without a word."""
    m, x = _module().eval(), torch.zeros(3, 1, 128)

    def run(c):
        with torch.no_grad():
            m(x, past_key_values=c)
    for length in (5, 6):
        c = _cache(dtype=torch.float32)
        c.begin([5, 5, 5])
        c.begin(1)
        at = c.position_ids.data_ptr()
        c.truncate(1, length)
        with pytest.raises(ValueError, match="begin"):
            run(c)
        c.begin(1)
        assert c.position_ids.data_ptr() == at               # a captured step reads them again
        with pytest.raises(RuntimeError, match="HIP device"):
            run(c)
    # a sequence that ends in front of a step takes no part in it, nor does one that takes none lose any
    c = _cache(dtype=torch.float32)
    c.begin([5, 5, 5])
    c.begin([1, 1, 0])
    c.free(0)
    c.truncate(2, 3)
    assert c.lengths.tolist() == [0, 6, 0] and c.new_tokens.tolist() == [0, 1, 0]
    with pytest.raises(RuntimeError, match="HIP device"):
        run(c)
