"""What kernels report about indices outside their tables reaches the callers
of Session and Answers, and what Answers refuses before it runs."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_check_device_raises_once(cuda):
    from sheaf_b200.runtime import ELEM_F32, ELEM_I32, Session, SheafB200Error

    s = Session(0)
    s.check_device()
    cache = s.kv_cache(2, 8, 1, 32, ELEM_F32)
    ints = lambda a: s.upload(np.asarray(a, np.int32), ELEM_I32)  # noqa: E731
    qkv = s.upload(np.ones((1, 3 * 32), np.float32))
    s.kv_append(cache, qkv, ints([0]), ints([3]), ints([[0, 1]]))
    s.check_device()
    s.kv_append(cache, qkv, ints([0]), ints([16]), ints([[0, 1]]))     # two pages hold 16
    with pytest.raises(SheafB200Error, match="outside"):
        s.check_device()
    s.check_device()
    s.prefix_attention(cache, s.upload(np.ones((1, 32), np.float32)), ints([17]), pages=ints([[0, 1]]))
    with pytest.raises(SheafB200Error, match="outside"):
        s.check_device()


def test_answers_ask(cuda):
    from sheaf_b200.runtime import SheafB200Error
    from tests.test_gpu_answers import _answers

    _, _, a = _answers("f32")
    a.draw([1, 2, 3], 2, 3)
    append = a.s.kv_append
    a.s.kv_append = lambda cache, qkv, seq, pos, pages, base=0: append(cache, qkv, seq, pos, pages, base + 1)
    with pytest.raises(SheafB200Error, match="outside"):  # the prompt's first token lies below its table
        a.draw([1, 2, 3], 2, 3)
    a.s.kv_append = append
    a.draw([1, 2, 3], 2, 3)


def test_answers_refuses_to_draw_from_nothing(cuda):
    from tests.test_gpu_answers import _answers

    _, _, a = _answers("f32")
    for k in (0, -1):
        with pytest.raises(ValueError):
            a.draw([1, 2, 3], 2, 3, k=k)
