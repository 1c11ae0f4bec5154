"""Session's cached-generation methods refuse buffers of another type or too
few values before anything reaches the device (buffers here have no memory)."""
import pytest

from sheaf_b200._lib import ELEM_BF16, ELEM_F32, ELEM_I32, KvCache
from sheaf_b200.runtime import ELEM_SIZE, Buffer, SheafB200Error, Session


class _Host(Session):
    def __init__(self):
        self._h = None

    def empty(self, shape, elem):
        raise AssertionError("nothing should have been refused")


class _Cache:
    desc = KvCache(0x10000, 0x20000, 8 * 2 * 64, 2 * 64, 64, 16, 8, 2, 64, ELEM_BF16)


def _buf(shape, elem):
    b, n = Buffer(None), 1
    for d in shape:
        n *= d
    b._meta = (tuple(shape), elem, n * ELEM_SIZE[elem])
    return b


def _refused(name, good, bad):
    s = _Host()
    with pytest.raises(AssertionError):  # the call as it should be goes through to the device
        getattr(s, name)(**good)
    with pytest.raises(SheafB200Error, match=name):
        getattr(s, name)(**{**good, **bad})


APPEND = dict(cache=_Cache, qkv=((5, 8 * 64), ELEM_BF16), seq=((5,), ELEM_I32), pos=((5,), ELEM_I32),
              pages=((3, 4), ELEM_I32), rotary=1, cos=((20, 32), ELEM_F32), sin=((20, 32), ELEM_F32))
ATTEND = dict(cache=_Cache, q=((6, 4 * 64), ELEM_BF16), lens=((3,), ELEM_I32), pages=((3, 4), ELEM_I32),
              prefix_pages=((1, 5), ELEM_I32), prefix_len=33)
SCORE = dict(logits=((4, 72), ELEM_F32), v=65, targets=((4,), ELEM_F32))
GRAD = dict(logits=((4, 72), ELEM_BF16), v=65, targets=((4,), ELEM_F32), dlogp=((4,), ELEM_F32),
            dentropy=((4,), ELEM_F32), scores=dict(lse=((4,), ELEM_F32), entropy=((4,), ELEM_F32)))


def _made(a):
    if isinstance(a, dict):
        return {k: _made(v) for k, v in a.items()}
    return _buf(*a) if isinstance(a, tuple) else a


@pytest.mark.parametrize("bad", [dict(qkv=((5, 8 * 64), ELEM_F32)), dict(qkv=((5, 8 * 64 + 8), ELEM_BF16)),
                                 dict(qkv=((5, 3 * 64), ELEM_BF16)), dict(qkv=((5 * 8 * 64,), ELEM_BF16)),
                                 dict(seq=((4,), ELEM_I32)), dict(pos=((5,), ELEM_F32)), dict(pos=((4,), ELEM_I32)),
                                 dict(pages=((12,), ELEM_I32)), dict(pages=((3, 4), ELEM_F32)), dict(cos=None),
                                 dict(sin=None), dict(sin=((19, 32), ELEM_F32)), dict(cos=((20, 32), ELEM_BF16))])
def test_append(bad):
    _refused("kv_append", _made(APPEND), _made(bad))


@pytest.mark.parametrize("bad", [dict(q=((6, 4 * 64), ELEM_F32)), dict(q=((6, 4 * 64 + 8), ELEM_BF16)),
                                 dict(q=((7, 4 * 64), ELEM_BF16)), dict(lens=((3,), ELEM_F32)),
                                 dict(lens=((0,), ELEM_I32)), dict(lens=((3, 1), ELEM_I32)),
                                 dict(pages=((2, 4), ELEM_I32)), dict(pages=((3, 4), ELEM_F32)),
                                 dict(prefix_pages=((4,), ELEM_I32)), dict(prefix_pages=((5,), ELEM_F32))])
def test_attention(bad):
    _refused("prefix_attention", _made(ATTEND), _made(bad))


@pytest.mark.parametrize("bad", [dict(logits=((4 * 72,), ELEM_F32)), dict(targets=((4,), ELEM_I32)),
                                 dict(targets=((3,), ELEM_F32))])
def test_logprobs(bad):
    _refused("token_logprobs", _made(SCORE), _made(bad))


@pytest.mark.parametrize("bad", [dict(targets=((4,), ELEM_I32)), dict(dlogp=((3,), ELEM_F32)),
                                 dict(dentropy=((4,), ELEM_BF16)), dict(logits=((288,), ELEM_BF16)),
                                 dict(scores=dict(lse=((3,), ELEM_F32), entropy=((4,), ELEM_F32))),
                                 dict(scores=dict(lse=((4,), ELEM_F32), entropy=((2, 1), ELEM_F32)))])
def test_logprobs_vjp(bad):
    _refused("token_logprobs_vjp", _made(GRAD), _made(bad))
