"""How near a chosen token is to the border of its share, and which launches a call makes."""
import pytest
import torch

from test_sample_gpu import BF16, F32, _logits, check

pytestmark = pytest.mark.gpu


def unit(vocab):
    """What a weight is a whole number of: 2^-50, or what the sums of a long row leave of 64 bits -- its weights, of at most 1, and one more."""
    frac = 50
    while (vocab + 1) << frac >= 1 << 64:
        frac -= 1
    return 2.0 ** -frac


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [2 ** 21 - 4, 262144, 131072, 128000, 40000])
def test_a_peak_and_a_flat_tail(vocab, dtype, dev):
    """A token of weight 1 and many of one small weight, which are all off in the same direction: by half a unit each, and by 2^-37 of themselves.  So is a sum by as much
    for each of its weights, of a total of 1 at least; a share by that twice, the log-probability once."""
    from odysseus_transformer_amd import ops
    d = 29.0
    falls = torch.arange(32.55, 47.0, 0.5, dtype=torch.float64)                      # the tail's weights are 2^-these
    temperature = (d / (falls * torch.log(torch.tensor(2.0, dtype=torch.float64)))).float()
    draws = torch.tensor([1 - 2 ** -24, 1 - 2 ** -23, 1 - 2 ** -20, 0.5, 0.0])
    for u in draws:
        x = torch.full((1, vocab), 1.0, dtype=dtype)
        x[0, vocab // 3] = 1.0 + d
        on = x.to(dev)
        for t in temperature:
            tokens, logs = (y.cpu() for y in ops.sample(on, u[None].to(dev), temperature=float(t)))
            w = torch.exp(torch.tensor(-d, dtype=torch.float64) / t.double())
            tail = (vocab - 1) * w
            total = 1 + tail
            off = (vocab - 1) * unit(vocab) / 2 + tail * 2 ** -37
            token = int(tokens[0])
            if token == vocab // 3:
                before, upto, log = 0.0, 1.0 / total, -torch.log1p(tail)
            else:
                rank = token + 1 if token < vocab // 3 else token                  # in the tail, from 1
                before, upto, log = (1 + (rank - 1) * w) / total, (1 + rank * w) / total, torch.log(w) - torch.log1p(tail)
            assert before - 2 * off <= float(u) <= upto + 2 * off, (vocab, float(t), float(u), token)
            # half a step of 32 bits; the power that the total's logarithm is corrected by is off by 2^-37 too
            assert abs(float(logs[0].double() - log)) <= off + 2 ** -24 * abs(float(log)) + 2 ** -36.5, (vocab, float(t), float(u), float(logs[0]), float(log))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [2 ** 16 - 1, 2 ** 17 - 2, 2 ** 17 - 1, 2 ** 17, 2 ** 20 - 1])
def test_sums_of_nearly_64_bits(vocab, dtype, dev):
    """Rows of equals, whose weights are all 1, and of infinite ones: their sums are the largest that a row of its length can have."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.99, 1 - 2 ** -24, 1.0])
    zeros = torch.zeros((6, vocab), dtype=dtype)
    for logits in (zeros, zeros + 3.5, zeros - 200.0, torch.full_like(zeros, float("inf"))):
        check(logits, u, dev)
        check(logits, u, dev, top_p=0.75)
        check(logits, u, dev, top_k=vocab - 1, min_p=1.0)


def _near_borders(steps, least, most, seed=1):
    """Rows of one token of 1 + 15/128 and `others` of 1.0, and a random number of 32 bits that is between 2^least and 2^most of the first one's share away from its border.
    (The two values lie at the ends of 16 that the kernel for bf16 forms weights of by 15 products with one factor.)"""
    g = torch.Generator().manual_seed(seed)
    n = 1 << 21
    others = torch.randint(50, 3000, (n,), generator=g).double()
    temperature = (0.3 + 1.2 * torch.rand((n,), generator=g)).float()
    border = 1 / (1 + others * torch.exp(-(steps / 128.0) / temperature.double()))
    u = border.float()
    away = (u.double() / border - 1).abs()
    those = ((away >= 2.0 ** least) & (away <= 2.0 ** most)).nonzero().flatten()[:400]
    return others[those].long(), temperature[those], u[those]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_borders_of_shares(dtype, dev):
    """Random numbers that are 2^-37 to 2^-35.5 of a share away from its border are on the side where 64 bits have them."""
    others, temperature, u = _near_borders(15, -37.0, -35.5)
    assert len(u) > 100
    logits = torch.full((len(u), 3000), -float("inf"))
    logits[:, 1:] = torch.where(torch.arange(2999)[None, :] < others[:, None], 1.0, -float("inf"))
    logits[:, 0] = 1.0 + 15 / 128
    check(logits.to(dtype), u, dev, temperature=temperature)


@pytest.mark.parametrize("rows,vocab,settings,sliced", [
    (1, 70000, dict(), True), (1, 70000, dict(top_p=0.9), True), (16, 70000, dict(top_p=0.9), True), (65, 70000, dict(), False), (1, 70000, dict(top_k=20), False),
    (1, 70000, dict(top_k=2049), False), (1, 65535, dict(), False), (3, 70000, dict(top_k="each"), True), (16, 70000, dict(top_k="each"), False), (16, 98304, dict(top_k="each"), True),
    (1, 98304, dict(top_k=20), True), (1, 98303, dict(top_k=2048), False), (1, 250000, dict(top_k=4000), False), (1, 250000, dict(top_k=250000), True),
    (1, 250000, dict(top_k=2 ** 31 - 1), True), (1, 250000, dict(temperature=0.0, top_k=4000), True), (1, 70000, dict(temperature=0.0), False),
    (2, 250000, dict(temperature="each", top_k=4000), False)], ids=str)
def test_which_rows_go_in_slices(rows, vocab, settings, sliced, dev):
    """Long fp32 rows: from 65536 logits on, from 98304 on where they are known to be read and little else, not with a top_k that slices can do nothing with."""
    from odysseus_transformer_amd import _lib, ops
    logits, u = _logits(rows, vocab, F32, seed=vocab)
    own = torch.arange(rows)
    given = {"top_k": (own % 3 * 30).to(torch.int32), "temperature": 1.0 - own % 2}
    settings = {k: given[k] if v == "each" else v for k, v in settings.items()}
    check(logits, u, dev, **settings)
    on = logits.to(dev), u.to(dev), {k: v.to(dev) if torch.is_tensor(v) else v for k, v in settings.items()}
    _lib.profile_enable(True)
    try:
        ops.sample(on[0], on[1], **on[2])
        torch.cuda.synchronize()
        launches = _lib.profile_collect()
    finally:
        _lib.profile_enable(False)
    assert ("sample_largest" in launches) == sliced and sum(n for n, _, _ in launches.values()) == (4 if sliced else 1), launches
