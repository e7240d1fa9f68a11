"""A cache in 8 bits to the byte: every value under every scale, rotated keys as the definition has them, tiles of 256 rows over pages of each size."""
import math

import pytest
import torch

import paged_q8_reference as q8
import paged_reference as ref
from paged_q8_reference import E8, F8
from test_paged_q8_gpu import _bytes, _check_heads, _inv_freq, _rows, _to

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_every_value_under_every_scale(D, dtype, dev):
    """Bytes of scale from 1 to 254: what the type has comes back exactly; below its smallest numbers the nearest one, half way to the even one, and beyond its largest an
    infinity, as conversions have it."""
    from odysseus_transformer_amd import ops
    page, block, Hkv = 64, 8, 4                                     # a block: 8 rows of 4 heads, all 254 values of one scale in each two heads or four
    pages = 32
    scales = (torch.arange(pages * 8) % 254 + 1).to(torch.uint8)    # 256 blocks
    values = torch.tensor([b for b in range(256) if b & 0x7f != 0x7f], dtype=torch.uint8)
    at = torch.arange(pages * page * Hkv * D).view(pages, page, Hkv, D)
    held = values[at % 254]
    k8, kz = held.to(dev).view(F8), scales.view(pages, 8, 1).expand(-1, -1, Hkv).contiguous().to(dev).view(E8)
    v8, vz = held.flip(0).contiguous().to(dev).view(F8), scales.flip(0).view(pages, 8, 1).expand(-1, -1, Hkv).contiguous().to(dev).view(E8)
    table, lengths = torch.arange(pages, dtype=torch.int32, device=dev)[None], torch.tensor([pages * page], dtype=torch.int32, device=dev)
    k, v = ops.paged_read_q8(k8, v8, kz, vz, table, lengths, pages * page, dtype)
    for have, b, z in ((k, held, scales), (v, held.flip(0), scales.flip(0))):
        exact = b.view(F8).double() * torch.exp2(z.double() - 127).view(pages, 8, 1, 1).repeat_interleave(block, 1)
        want = exact.float().to(dtype)                              # 32 bits hold them all, but for those beyond the largest
        assert torch.equal(have.cpu().view(-1), want.view(-1))
        fits = (exact % 2.0 ** (-133 if dtype == BF16 else -149) == 0) & (exact.abs() < 2.0 ** 128)
        assert torch.equal(have.double().cpu().view(-1)[fits.view(-1)], exact.view(-1)[fits.view(-1)]) and bool((~fits).any())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_ends_of_what_is_appended(dtype, dev):
    """The smallest scale that append writes, and the largest: the nearest of eight bits to a number from 1.9375 * 2^127 on is 2^128, which is infinite when it is read."""
    from odysseus_transformer_amd import ops
    D, page = 64, 16
    c = q8.make([16, 16, 16], 16, 1, 1, D, page, 16, dtype, seed=1)
    x = torch.zeros((3, 16, 3, D))
    x[0, :, 2] = 2.0 ** -130 * torch.arange(16).view(16, 1)
    x[1, 0, 2, :3] = torch.tensor([1.75 * 2.0 ** 127, 1.875 * 2.0 ** 127, -1.875 * 2.0 ** 127])
    x[2, 0, 2, :2] = torch.tensor([1.984375 * 2.0 ** 127, 2.0 ** 127])
    g = _to(c, dev)
    ops.paged_append_q8_(x.to(dtype).to(dev), 1, *q8.cache(g), rotate=False)
    assert [int(g["vz"].view(torch.uint8)[c["table"][s, 0].item(), 0, 0]) for s in range(3)] == [1, 247, 247]
    v = ops.paged_read_q8(*q8.cache(g), 16, F32)[1].cpu()
    assert torch.equal(v[0, :, 0, 0], x[0, :, 2, 0])               # sixteenths of the scale below 1 have four bits
    assert v[1, 0, 0, :3].tolist() == [1.75 * 2.0 ** 127, 1.875 * 2.0 ** 127, -1.875 * 2.0 ** 127] and v[2, 0, 0, :2].tolist() == [math.inf, 2.0 ** 127]


@pytest.mark.parametrize("n,H,D,dtype", [(1, 2, 128, BF16), (1, 2, 64, BF16), (70, 32, 128, BF16), (70, 32, 64, BF16), (256, 64, 128, BF16), (3, 2, 64, F32)], ids=lambda x: str(x)[-4:])
@pytest.mark.parametrize("byte", [1, 2, 3, 10])
def test_attention_over_the_smallest_scales(byte, n, H, D, dtype, dev):
    """Values down to 2^-135: what is below the type's smallest normal number takes part, rounded to its smallest one of all."""
    from odysseus_transformer_amd import ops
    c = q8.make([300], n, H, H, D, 16, 8, dtype, seed=1)
    z = c["vz"].view(torch.uint8)
    z.copy_(torch.where(z == 255, 255, torch.full_like(z, byte)))
    held = c["v8"].double()
    c["v"] = torch.where(torch.isnan(held), 0.0, held) * 2.0 ** (byte - 127 + 100)      # bounds are reckoned 2^100 higher
    g = _to(c, dev)
    out, _ = ops.paged_attn_q8(g["q"], *q8.cache(g))
    part = dict(c, q=c["q"][:, :, :1], k=c["k"][:, :, :1], v=c["v"][:, :, :1])
    o, s, mean, dots = ref.attend(part)
    # beside them half a step of the smallest numbers for the values and for the result
    least = 2.0 ** (-133 + 100) if dtype == BF16 else 2.0 ** (-149 + 100)
    assert ((out[:, :, :1].double().cpu() * 2.0 ** 100 - o).abs() <= ref.attend_bounds(part, o, s, mean, dots)[0] + least).all()


@pytest.mark.parametrize("D,page,block", [(128, 16, 16), (128, 64, 64), (128, 64, 32), (128, 8, 8), (128, 128, 64)])
def test_tiles_of_256_rows_over_pages_of_each_size(D, page, block, dev):
    """Row tiles of 256, of 64 (sequence, kv head) pairs, which the workspace's size shows: a scale for a whole tile of keys, for half of one, for a group of eight."""
    from odysseus_transformer_amd import _lib
    lengths, n, H = [256 + 64, 300, 517, 64, 191, 1, 0, 256 + 65], 256, 8
    c = q8.make(lengths, n, H, H, D, page, block, BF16, seed=page)
    c["table"][2, 1] = -1
    width = c["table"].shape[1]
    parts = _lib.load().ody_paged_attn_q8_workspace_bytes(len(lengths), n, H, H, D, page, width, 0)
    assert parts == 256 * 2 * 256 * (D * 4 + 8)                    # 256 blocks, two units each, of 256 rows
    _check_heads(c, _to(c, dev), dev, (0, 5))


@pytest.mark.parametrize("D,page,block", [(64, 16, 16), (64, 64, 64), (64, 8, 8)])
def test_tiles_of_128_rows_of_heads_of_64(D, page, block, dev):
    from odysseus_transformer_amd import _lib
    lengths, n, H = [200, 128, 321, 130, 64, 191, 1, 0], 128, 8
    c = q8.make(lengths, n, H, H, D, page, block, BF16, seed=page)
    parts = _lib.load().ody_paged_attn_q8_workspace_bytes(len(lengths), n, H, H, D, page, c["table"].shape[1], 0)
    assert parts % (2 * 128 * (D * 4 + 8)) == 0 and parts // (2 * 128 * (D * 4 + 8)) == 512
    _check_heads(c, _to(c, dev), dev, (0, 5))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lengths,n,D,block", [([100, 37, 64], 1, 128, 32), ([300, 131, 70], 67, 128, 16), ([700, 513], 500, 64, 64), ([2100], 2100, 128, 8)], ids=str)
def test_rotated_keys_to_the_byte(lengths, n, D, block, dtype, dev):
    """The angle is the 32-bit product; its cosine and sine, of 64 bits, are rounded to 32 and then to the type; the rotated key is rounded to 32 bits and then to eight.  (Where 64
    bits of a cosine come out a last place apart on two machines, one in 2^28 of those of 32 bits differs.)"""
    from odysseus_transformer_amd import ops
    Hq, Hkv, page = 3, 3, 64
    c = q8.make(lengths, n, Hq, Hkv, D, page, block, dtype, seed=n)
    g, f = _to(c, dev), _inv_freq(D)
    x, half = c["qkv"], D // 2
    place = torch.tensor(lengths)[:, None] - n + torch.arange(n)
    th = (place.clamp(min=0).float()[:, :, None] * f).double()
    cos, sin = (t(th).float().to(dtype).double()[:, :, None] for t in (torch.cos, torch.sin))
    keys = x[:, :, Hq:Hq + Hkv].double()
    a, b = keys[..., :half], keys[..., half:]
    c["qkv"] = x.double()
    c["qkv"][:, :, Hq:Hq + Hkv] = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    # as they are: rounded to 32 bits, then to eight
    _, (k_rows, k_scales, _, _), (v_rows, v_scales, _) = q8.append(c, Hq)
    ops.paged_append_q8_(x.to(dev), Hq, *q8.cache(g), inv_freq=f.to(dev))
    assert torch.equal(_bytes(g["kz"]), k_scales) and torch.equal(_bytes(g["vz"]), v_scales)
    assert torch.equal(_rows(g["k8"]), _rows(k_rows)) and torch.equal(_rows(g["v8"]), _rows(v_rows))
