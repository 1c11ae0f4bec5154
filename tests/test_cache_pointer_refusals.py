"""Pointers that are not on whole values, and memory that would be read and
written in two layouts at once, are refused on the host (nothing is read)."""
import pytest

from tests.test_cache_refusals import ARGS, BF16, F32, P, _append, _attend, _cache, _grad, _score
from tests.test_cache_refusals import L  # noqa: F401  (fixture)


@pytest.mark.parametrize("change", [dict(qkv=P + 1), dict(q_out=2 * P + 1), dict(seq=P + 2), dict(pos=P + 1),
                                    dict(pages=P + 3), dict(cos=P + 2), dict(sin=P + 1)])
def test_append_wants_whole_values(L, change):  # noqa: F811
    assert _append(L, **{**dict(q_out=2 * P), **change}) == ARGS


def test_append_of_f32_wants_whole_values(L):  # noqa: F811
    for change in (dict(qkv=P + 2, q_out=2 * P), dict(q_out=2 * P + 2)):
        assert _append(L, _cache(elem=F32), **change) == ARGS


def test_append_in_place_wants_one_stride(L):  # noqa: F811
    assert _append(L, qkv=P, q_out=P, ldq=256) == ARGS


@pytest.mark.parametrize("change", [dict(lse=P + 2), dict(prefix_pages=P + 2), dict(pages=P + 1), dict(lens=P + 3)])
def test_attention_wants_whole_values(L, change):  # noqa: F811
    assert _attend(L, **change) == ARGS


@pytest.mark.parametrize("name", ["targets", "logp", "entropy", "lse", "ids", "alt"])
def test_logprobs_wants_whole_values(L, name):  # noqa: F811
    assert _score(L, **{name: P + 2}) == ARGS


@pytest.mark.parametrize("name", ["targets", "lse", "entropy", "dlogp", "dentropy"])
@pytest.mark.parametrize("elem", [BF16, F32])
def test_logprobs_vjp_wants_whole_values(L, name, elem):  # noqa: F811
    assert _grad(L, elem=elem, **{name: P + 2}) == ARGS
