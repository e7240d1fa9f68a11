"""What the entry points of a cache in pages accept at the limits of their index arithmetic.  Nothing is launched: a call that passes the check in
question is refused by a later one."""
import pytest

from odysseus_transformer_amd import _lib

Q = 16            # an aligned address that nothing is read from
LIMIT = 2 ** 31 - 4096


def _code(name, S=1, n=1, Hq=4, Hkv=2, D=64, pages=4, page=16, width=3, dtype=0):
    """The status of a call whose pages are misaligned (-3, the last of the checks that both share)."""
    xs, ps = (512, 512, 64), (1 << 20, 130, 64)
    with pytest.raises(_lib.OdysseusHipError) as e:
        if name == "ody_paged_append":
            _lib.call(name, Q, Q, Q, Q, Q, Q, 0, 0, Q, S, n, Hq, Hkv, D, *xs, *xs, *ps, *ps, pages, page, width, width, dtype, 0)
        else:
            _lib.call(name, Q, Q, Q, Q, Q, 0, Q, Q, S, n, Hq, Hkv, D, *xs, *ps, *ps, *xs, pages, page, width, width, 1.0, dtype, 0, 0, 0)
    return e.value.code


@pytest.mark.parametrize("name", ["ody_paged_append", "ody_paged_attn"])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 2048, 4096, 1 << 14])
def test_room_behind_the_last_column(name, page):
    """Attention looks up the pages of tiles to come before it knows that there are none; places behind the table's last column have to be numbers of 31 bits."""
    most = LIMIT // page
    assert _code(name, page=page, width=most) == -3
    assert _code(name, page=page, width=most + 1) == -1
    assert _code(name, page=page, width=2 ** 31 // page - 1) == (-3 if most == 2 ** 31 // page - 1 else -1)


@pytest.mark.parametrize("name", ["ody_paged_append", "ody_paged_attn"])
def test_new_tokens_and_heads(name):
    """Rows, and vectors of a token, are counted in 32 bits; the products that the check forms fit 64 whatever the sizes are."""
    top = 2 ** 31 - 1
    for sizes in (dict(S=top, n=top, Hq=2, Hkv=1), dict(S=top, n=top, Hq=top, Hkv=1), dict(S=top, n=3, Hq=top, Hkv=top), dict(S=1 << 29, n=1, Hq=2, Hkv=1),
                  dict(n=1 << 29, Hq=2, Hkv=1), dict(n=2 ** 31 // 6, Hq=4, Hkv=1), dict(Hq=2 ** 27, Hkv=1), dict(Hq=top, Hkv=1), dict(Hq=2 ** 30, Hkv=2 ** 30)):
        assert _code(name, **sizes) == -1, sizes
    for sizes in (dict(S=1 << 28, n=1, Hq=4, Hkv=1), dict(n=2 ** 31 // 6 - 64, Hq=4, Hkv=1), dict(Hq=2 ** 26, Hkv=1)):
        assert _code(name, **sizes) == -3, sizes


def test_tokens_of_one_launch():
    """A block of 256 threads for a token, and fewer than 2^32 threads in a launch: refused by name, and before anything is launched."""
    for S, n, code in ((1 << 14, 1 << 10, -1), (1 << 24, 1, -1), (1 << 12, (1 << 12) - 1, -3)):
        with pytest.raises(_lib.OdysseusHipError) as e:   # -3: the projection is misaligned
            _lib.call("ody_paged_append", Q, Q, Q, Q, Q, Q, 0, 0, Q, S, n, 2, 1, 64, 256, 256, 60, 128, 128, 64, 2048, 64, 64, 2048, 64, 64, 4, 16, 3, 3, 0, 0)
        assert e.value.code == code, (S, n)
