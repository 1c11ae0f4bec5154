"""What the cached-generation entry points refuse, and with which code: all of
it is decided on the host before any GPU work (pointers here are never read)."""
import ctypes as C

import pytest

BF16, F32, F16 = 0x22000010, 0x21000020, 0x21000010
ARGS, ALIGN, WORKSPACE = 1, 2, 5
P = 0x10000  # an aligned address that is never read


@pytest.fixture(scope="module")
def L():
    import sheaf_b200

    return sheaf_b200.lib()


def _cache(**change):
    from sheaf_b200 import KvCache

    f = dict(k=P, v=P, page_stride=16 * 2 * 64, row_stride=2 * 64, head_stride=64, n_pages=8, page_rows=16, n_heads=2,
             head_dim=64, elem=BF16)
    f.update(change)
    return KvCache(**f)


BAD_CACHES = [(dict(elem=F16), ARGS), (dict(head_dim=48), ARGS), (dict(head_dim=256), ARGS), (dict(n_heads=0), ARGS),
              (dict(page_rows=0), ARGS), (dict(n_pages=-1), ARGS), (dict(k=0), ARGS), (dict(row_stride=-128), ARGS),
              (dict(page_stride=1 << 41), ARGS), (dict(k=P + 2), ALIGN), (dict(row_stride=130), ALIGN),
              (dict(head_stride=68), ALIGN)]


def _append(L, cache=None, **change):
    a = dict(qkv=P, ld=(4 + 4) * 64, n=3, h_q=4, q_out=P, ldq=256, seq=P, pos=P, base=0, pages=P, n_seqs=2, max_pages=4,
             rotary=1, rot_dim=64, cos=P, sin=P, n_pos=64)
    a.update(change)
    return L.sb_op_kv_append(cache if cache is not None else _cache(), *a.values(), None)


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_cache_descriptions(L, change, code):
    bad = _cache(**change)
    assert _append(L, bad) == code
    assert _attend(L, bad) == code
    assert L.sb_op_prefix_attention_workspace_size(bad, 2, 1, 4, 64, 4) == 0


@pytest.mark.parametrize("change", [dict(qkv=None), dict(ld=511), dict(n=-1), dict(h_q=-1), dict(q_out=None),
                                    dict(ldq=255), dict(seq=None), dict(pos=None), dict(base=-1), dict(pages=None),
                                    dict(rotary=3), dict(rotary=-1), dict(rot_dim=0), dict(rot_dim=7),
                                    dict(rot_dim=66), dict(cos=None), dict(sin=None), dict(n_pos=0),
                                    dict(max_pages=-1), dict(n_seqs=-1)])
def test_append_refuses(L, change):
    assert _append(L, **change) == ARGS


def test_append_of_nothing_is_done(L):
    assert _append(L, n=0) == 0
    assert L.sb_op_kv_append(None, P, 512, 1, 4, P, 256, P, P, 0, P, 2, 4, 0, 0, None, None, 0, None) == ARGS


def _attend(L, cache=None, **change):
    a = dict(q=P, ldq=256, out=P, ldo=256, lse=None, b=2, tq=1, h_q=4, scale=0.125, prefix_pages=P, prefix_len=64,
             pages=P, max_pages=4, lens=P, workspace=P, size=1 << 40)
    a.update(change)
    return L.sb_op_prefix_attention(cache if cache is not None else _cache(), *a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), ARGS), (dict(out=None), ARGS), (dict(lens=None), ARGS), (dict(ldq=255), ARGS), (dict(ldo=128), ARGS),
    (dict(ldq=260), ALIGN), (dict(ldo=258), ALIGN), (dict(q=P + 8), ALIGN), (dict(out=P + 2), ALIGN),
    (dict(b=-1), ARGS), (dict(tq=-1), ARGS), (dict(h_q=0), ARGS), (dict(h_q=3), ARGS), (dict(scale=0.0), ARGS),
    (dict(scale=-1.0), ARGS), (dict(scale=float("nan")), ARGS), (dict(scale=float("inf")), ARGS),
    (dict(prefix_pages=None), ARGS), (dict(prefix_len=-1), ARGS), (dict(pages=None), ARGS), (dict(max_pages=-1), ARGS),
    (dict(max_pages=1 << 27), ARGS), (dict(b=1 << 15, tq=1 << 15), ARGS)])
def test_attention_refuses(L, change, code):
    assert _attend(L, **change) == code


def test_attention_wants_its_workspace(L):
    need = L.sb_op_prefix_attention_workspace_size(_cache(), 2, 1, 4, 64, 4)
    assert need > 0
    assert _attend(L, workspace=None) == WORKSPACE
    assert _attend(L, size=need - 1) == WORKSPACE
    assert _attend(L, workspace=P + 4) == WORKSPACE
    assert _attend(L, cache=_cache(n_pages=0), prefix_len=64) == ARGS


def test_attention_of_nothing_is_done(L):
    assert _attend(L, b=0) == 0
    assert _attend(L, tq=0) == 0


def _score(L, **change):
    a = dict(elem=BF16, x=P, ld=100, rows=4, v=100, targets=P, temperature=1.0, logp=P, entropy=P, lse=P, k=5, ids=P,
             alt=P)
    a.update(change)
    return L.sb_op_token_logprobs(*a.values(), None)


@pytest.mark.parametrize("change", [dict(elem=F16), dict(x=None), dict(ld=99), dict(rows=-1), dict(v=0), dict(v=-3),
                                    dict(targets=None), dict(temperature=0.0), dict(temperature=-1.0),
                                    dict(temperature=float("nan")), dict(temperature=float("inf")), dict(k=-1),
                                    dict(k=33), dict(v=4, k=5), dict(x=P + 1), dict(ld=1 << 41)])
def test_logprobs_refuses(L, change):
    assert _score(L, **change) == ARGS


def _grad(L, **change):
    a = dict(elem=F32, x=P, ld=100, rows=4, v=100, targets=P, temperature=1.0, lse=P, entropy=P, dlogp=P, dentropy=P,
             dx=2 * P, ldd=100)
    a.update(change)
    return L.sb_op_token_logprobs_bwd(*a.values(), None)


@pytest.mark.parametrize("change", [dict(elem=F16), dict(x=None), dict(dx=None), dict(lse=None), dict(targets=None),
                                    dict(entropy=None), dict(ld=99), dict(ldd=99), dict(rows=-1), dict(v=0),
                                    dict(temperature=0.0), dict(x=P + 2), dict(dx=P, ldd=104)])
def test_logprobs_vjp_refuses(L, change):
    assert _grad(L, **change) == ARGS


def test_scores_of_no_rows_are_done(L):
    assert _score(L, rows=0) == 0
    assert _grad(L, rows=0) == 0
    assert C.sizeof(_cache()) == 64  # as the C struct lays it out
