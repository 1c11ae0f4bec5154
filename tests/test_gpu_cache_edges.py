"""Corners of cached generation and scoring: idle slots, NaN and infinities,
logits and scores far from zero, pointers at odd places. Plain restatements
and tolerances as in test_gpu_cache.py."""
import numpy as np
import pytest

from tests.test_gpu_cache import ELEM, U, _Attend, _attend64, _cache, _check_attention, _f64, _i, _stream, _t

pytestmark = pytest.mark.gpu


def _check_rows(a, got, lse, rows):
    """Rows (sequence, query) of a call's results against float64."""
    q, k, v = (_f64(x) for x in (a.q, a.k, a.v))
    for s, t in rows:
        r = s * a.tq + t
        n = a.lens[s] - a.tq + t + 1 if a.lens[s] >= 0 else -1
        one = _attend64(q[r:r + 1, :a.hq * a.hd], k, v, a.prefix_table, a.prefix, a.table[s:s + 1], [n], 1, a.scale,
                        a.page)
        _check_attention(a.kind, got[r:r + 1], lse[r:r + 1], one, a.hd)


# ---- attention: idle slots -----------------------------------------------------


@pytest.mark.parametrize("hq,hkv,hd,prefix,idle", [(12, 12, 64, 1000, 128), (8, 4, 128, 700, 64), (6, 6, 32, 1500, 192)])
def test_f32_attention_beside_many_idle_slots(hq, hkv, hd, prefix, idle, cuda):
    """Whole tiles of rows that see nothing, whose queries (NaN) must not take the place of the next tile's."""
    import torch

    lens = ([3] * 64 + [-1] * idle) * 2 + [5] * 40
    a = _Attend("f32", hq, hkv, hd, 16, prefix, lens, 1, cuda)
    a.q[torch.from_numpy(a.lens < 0).to(cuda)] = float("nan")
    got, lse = a()
    live = a.lens >= 0
    assert (got[~live] == 0).all() and np.isneginf(lse[~live]).all()
    edge = 64 + idle
    _check_rows(a, got, lse, [(s, 0) for s in (0, 63, edge, edge + 1, edge + 63, 2 * edge, len(lens) - 1)])
    assert np.isfinite(got).all() and np.isfinite(lse[live]).all()
    first, first_lse = a.out.clone(), a.lse.clone()
    for _ in range(20):
        a()
        assert torch.equal(a.out, first) and torch.equal(a.lse, first_lse)


# ---- append: tables at odd places ------------------------------------------------


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("mode", [1, 2])
def test_append_with_angles_at_any_float(kind, mode, cuda):
    """Tables that start 4, 1 and 8 floats into an allocation give what tables at its start give."""
    import torch
    import sheaf_b200 as sb

    hq, hkv, hd, n = 8, 2, 64, 33
    width, g = (hq + 2 * hkv) * hd, torch.Generator().manual_seed(mode)
    qkv = torch.randn(n, width, generator=g).to(torch.float32 if kind == "f32" else torch.bfloat16).to(cuda)
    ang = torch.randn(n, hd // 2, generator=g)
    table, seq, pos = (_i(x, cuda) for x in (np.arange(3)[None], np.zeros(n), np.arange(n)))
    want = None
    for shift in (0, 4, 1, 8):
        cs = torch.zeros(2, shift + ang.numel(), device=cuda)
        cs[0, shift:], cs[1, shift:] = ang.cos().flatten().to(cuda), ang.sin().flatten().to(cuda)
        rows = [cs[i].clone() for i in range(2)]  # allocations of their own
        k, v = (torch.zeros(3, 16, hkv, hd, device=cuda, dtype=qkv.dtype) for _ in range(2))
        q = torch.zeros(n, hq * hd, device=cuda, dtype=qkv.dtype)
        assert sb.lib().sb_op_kv_append(_cache((k, v)), qkv.data_ptr(), width, n, hq, q.data_ptr(), hq * hd,
                                        seq.data_ptr(), pos.data_ptr(), 0, table.data_ptr(), 1, 3, mode, hd,
                                        rows[0][shift:].data_ptr(), rows[1][shift:].data_ptr(), n, _stream()) == 0
        if want is None:
            want = q, k, v
            assert q.abs().max() > 0 and k.abs().max() > 0
        assert all(torch.equal(x, y) for x, y in zip((q, k, v), want))


# ---- attention: rows that are zero whatever the cache holds ------------------------


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd,prefix", [(2, 2, 64, 40), (2, 2, 64, 20), (8, 1, 128, 30), (1, 1, 32, 64),
                                              (8, 1, 64, 64), (8, 1, 32, 32), (80, 1, 64, 64)])
def test_idle_rows_stay_zero_beside_infinite_values(kind, hq, hkv, hd, prefix, cuda):
    """Nothing but a short prefix, one part: idle slots share a tile of rows with slots that see an infinite value."""
    a = _Attend(kind, hq, hkv, hd, 16, prefix, [0, -1, 0, -1, 0], 1, cuda)
    assert a.table.shape[1] == 0
    for bad in (float("inf"), float("nan"), float("-inf")):
        a.v[int(a.prefix_table[0]), 3, :, 7] = bad
        got, lse = a()
        idle = a.lens < 0
        assert (got[idle] == 0).all() and np.isneginf(lse[idle]).all()
        assert not np.isfinite(got[~idle][..., 7]).any() and np.isfinite(np.delete(got[~idle], 7, 2)).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("slots", [3, 9, 80])
def test_rows_without_a_finite_score_are_zero(kind, slots, cuda):
    """All scores are -inf, and a value that the rows see is infinite."""
    a = _Attend(kind, 2, 2, 64, 16, 30, [0] * slots, 1, cuda)
    a.q[..., ::64] = 1.0
    a.k[..., 0] = float("-inf")
    a.v[int(a.prefix_table[0]), 5, :, 9] = float("inf")
    got, lse = a()
    assert (got == 0).all() and np.isneginf(lse).all()


# ---- attention: NaN is not hidden ----------------------------------------------------


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd,prefix,lens", [(2, 2, 64, 40, [3, 2]), (8, 2, 128, 300, [5] * 9),
                                                   (4, 4, 64, 2000, [40] * 80)])
def test_nan_queries_and_keys_show(kind, hq, hkv, hd, prefix, lens, cuda):
    """A NaN query's row is NaN and no other; so is every row that sees a NaN key, the first of all or its only one."""
    a = _Attend(kind, hq, hkv, hd, 16, prefix, lens, 1, cuda)
    clean, clean_lse = a()
    q = a.q.clone()
    a.q[1, 5] = float("nan")            # head 0 of sequence 1
    got, lse = a()
    assert np.isnan(got[1, 0]).all() and np.isnan(lse[1, 0])
    got[1, 0], lse[1, 0] = clean[1, 0], clean_lse[1, 0]
    assert np.array_equal(got, clean) and np.array_equal(lse, clean_lse)
    a.q.copy_(q)
    a.k[int(a.table[0][0]), 0] = float("nan")  # the first of sequence 0's own keys
    got, lse = a()
    assert np.isnan(got[0]).all() and np.isnan(lse[0]).all()
    assert np.array_equal(got[1:], clean[1:]) and np.array_equal(lse[1:], clean_lse[1:])
    a.k[int(a.prefix_table[0])] = float("nan")  # the first keys of all
    got, lse = a()
    assert np.isnan(got).all() and np.isnan(lse).all()
    a.prefix, a.lens = 0, np.ones_like(a.lens)   # its own first key alone
    got, lse = a()
    assert np.isnan(got[0]).all() and np.isnan(lse[0]).all()
    assert np.isfinite(got[1:]).all() and np.isfinite(lse[1:]).all()


# ---- log probabilities far from zero ----------------------------------------------------


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,v,k", [(40, 40, 8), (40, 1031, 20), (40, 5000, 8), (400, 9001, 5), (400, 40000, 0)])
@pytest.mark.parametrize("temperature", [1e-6, 1.0, 1e6])
def test_logprobs_of_large_logits(kind, rows, v, k, temperature, cuda):
    """Logits far from zero, whose ratio to the temperature leaves no bits behind its point in float32."""
    import torch
    import sheaf_b200 as sb

    rng = np.random.default_rng(v)
    at = np.array([3e3, 2e4, 1e6, 8657043456.0, 1e10, -1e10, 1e20, -1e20, 1e28, -3e37, 3e37, -7e3, 0.0, 4.2e6, 8.5e6,
                   -8.5e6, 1.7e7, 2.0 ** 31, -2.0 ** 33, 3003.0])
    s = at[np.arange(rows) % len(at)][:, None]
    x = s + np.abs(s) * 2.0 ** -7 * rng.standard_normal((rows, v)) + rng.standard_normal((rows, v))
    x[::2, v // 3] = x[::2].max(1)                                   # two equal largest ones
    x[::3, : v // 2] = -np.inf
    x[::5] = s[::5]                                                  # all equal
    xd = torch.from_numpy(x.astype(np.float32)).to(torch.float32 if kind == "f32" else torch.bfloat16).to(cuda)
    x64 = _f64(xd)
    t = np.where(np.arange(rows) % 2 == 0, x64.argmax(1), rng.integers(0, v, rows)).astype(np.float32)
    td = torch.from_numpy(t).to(cuda)
    logp, ent, lse, alt = (torch.full(n, 9.0, device=cuda) for n in ((rows,), (rows,), (rows,), (rows, max(k, 1))))
    ids = torch.full((rows, max(k, 1)), -9, device=cuda, dtype=torch.int32)
    assert sb.lib().sb_op_token_logprobs(ELEM[kind], xd.data_ptr(), v, rows, v, td.data_ptr(), temperature,
                                         logp.data_ptr(), ent.data_ptr(), lse.data_ptr(), k, ids.data_ptr(),
                                         alt.data_ptr(), _stream()) == 0
    big = float(np.finfo(np.float32).max)
    as_f32 = lambda a: np.where(a > big, np.inf, np.where(a < -big, -np.inf, a))  # noqa: E731
    z = x64 / float(np.float32(temperature))
    m = z.max(1, keepdims=True)
    log_sum = np.log(np.exp(z - m).sum(1, keepdims=True))
    lp = (z - m) - log_sum
    with np.errstate(invalid="ignore"):
        ent64 = -np.where(np.exp(lp) > 0, np.exp(lp) * lp, 0).sum(1)
    at_t = np.take_along_axis(lp, t.astype(int)[:, None], 1)[:, 0]
    # the arithmetic's bounds as in test_logprobs: few roundings of each result and, for lse, of the largest z
    for got, want, size in ((lse, (m + log_sum)[:, 0], np.abs(m[:, 0])), (logp, at_t, np.zeros(rows))):
        got, want = _f64(got), as_f32(want)
        assert np.array_equal(np.isinf(got), np.isinf(want)) and not np.isnan(got).any()
        ok = np.isfinite(want)
        assert (got[~ok] == want[~ok]).all()
        w = np.abs(want[ok])
        assert (np.abs(got[ok] - want[ok]) <= 1e-6 + 256 * U * w.clip(0, 1) + 4 * U * (w + size[ok])).all()
    assert (np.abs(_f64(ent) - ent64) <= 256 * U * np.maximum(ent64, 0.05)).all()
    if k:
        best = np.argsort(-x64, axis=1, kind="stable")[:, :k]
        assert np.array_equal(ids.cpu().numpy(), best)
        a64, a = as_f32(np.take_along_axis(lp, best, 1)), _f64(alt)
        assert np.array_equal(np.isneginf(a), np.isneginf(a64))
        ok = np.isfinite(a64)
        assert (np.abs(a[ok] - a64[ok]) <= 1e-6 + 16 * U * (1 + np.abs(a64[ok]))).all()


# ---- attention: infinite and NaN values in every kernel -----------------------------------

BAD_VALUES = [
    # kind, hq, hkv, hd, page, prefix, lens, tq: what the rows see ends inside tiles
    ("bf16", 6, 2, 64, 16, 200, [20, 33, -1, 7], 1),           # a warp: 12 rows behind the prefix, 3 own ones
    ("bf16", 4, 4, 128, 16, 200, [20] * 7 + [9], 3),           # 4 warps, 128 values: 24 rows
    ("bf16", 2, 2, 128, 12, 300, [61, 7] * 9, 3),              # 4 warps, pages of 12: 54 rows
    ("bf16", 1, 1, 64, 20, 500, [90, 41, 120], 40),            # 4 warps, pages of 20: 120 rows, several row tiles
    ("bf16", 4, 1, 64, 16, 600, [130, 5, -1, 64], 30),         # tcgen05: prefix of 480 rows, own 120
    ("bf16", 4, 4, 32, 24, 2000, [40, 3] * 50, 1),             # tcgen05: 100 rows, key tiles dealt out
    ("bf16", 4, 2, 128, 64, 5000, [129, 200, 70], 40),         # tcgen05: 240 rows, own 80
    ("bf16", 8, 1, 64, 8, 0, [1000, 257], 37),                 # own keys alone, 296 rows
    ("bf16", 1, 1, 128, 16, 13000, [500], 24),                 # tcgen05: 24 rows, key tiles dealt out; own on 4 warps
    ("f32", 6, 2, 64, 16, 200, [20, 33, -1, 7], 1),
    ("f32", 4, 4, 128, 16, 300, [20] * 7 + [9], 3),
    ("f32", 4, 1, 64, 24, 600, [130, 5, -1, 64], 30),
]


@pytest.mark.parametrize("kind,hq,hkv,hd,page,prefix,lens,tq", BAD_VALUES)
def test_attention_infinite_values_reach_those_that_see_them(kind, hq, hkv, hd, page, prefix, lens, tq, cuda):
    """Infinities and NaN in values: first in keys that only some queries see, then behind every query's last key, then
    in the shared prefix. A column of a row is then NaN or infinite where the row sees such a key, and otherwise bit for
    bit what it was; and the call repeats itself."""
    import torch

    a = _Attend(kind, hq, hkv, hd, page, prefix, lens, tq, cuda, capacity=max(lens) + page)
    lens = np.array(lens)
    clean, clean_lse = a()
    group = hq // hkv
    hit = np.zeros(clean.shape, bool)

    def spoil(table, j, head, col, x, rows):
        a.v[int(table[j // page]), j % page, head, col] = x
        hit[rows, head * group:(head + 1) * group, col] = True

    def check():
        got, lse = a()
        assert np.array_equal(got[~hit], clean[~hit]) and not np.isfinite(got[hit]).any()
        assert np.array_equal(lse, clean_lse)
        first = a.out.clone()
        for _ in range(3):
            a()
            assert torch.equal(a.out.view(torch.uint8), first.view(torch.uint8))

    for s in np.nonzero(lens >= 0)[0]:
        n = lens[s]
        # behind the end: nobody sees it
        for j in range(n, min(n + 3, a.table.shape[1] * page)):
            spoil(a.table[s], j, hkv - 1, j % hd, float("nan"), [])
        # the last key (the last query's own) and an earlier one among the queries' own
        for j, col, x in ((n - 1, 1, float("inf")), (n - tq // 2 - 1, 2, float("nan")), (n - tq, 3, float("-inf")),
                          (n // 3, 4, float("inf"))):
            if 0 <= j < n:
                spoil(a.table[s], j, s % hkv, (col * 7 + s) % hd, x,
                      [s * tq + t for t in range(tq) if n - tq + t >= j])
    check()
    if prefix:
        # behind the prefix's end, and inside, where short sequences with several queries stop before it
        for j in range(prefix, min(prefix + 2, len(a.prefix_table) * page)):
            a.v[int(a.prefix_table[j // page]), j % page, 0, 5] = float("inf")
        check()
        for j, col, x in ((prefix - 1, 11, float("nan")), (prefix - max(tq - 2, 1), 12, float("inf")),
                          (prefix // 2, 13, float("-inf"))):
            spoil(a.prefix_table, j, 0, col, x,
                  [s * tq + t for s in np.nonzero(lens >= 0)[0] for t in range(tq) if prefix + lens[s] - tq + t >= j])
            check()


@pytest.mark.parametrize("hd,seqs,prefix,key", [(64, 50, 2000, 1990), (128, 50, 2000, 1990), (64, 50, 1900, 1800),
                                                (32, 50, 2000, 1990)])
def test_attention_value_counts_once_where_key_tiles_are_dealt(hd, seqs, prefix, key, cuda):
    """tcgen05, one row tile whose key tiles two groups of warps take in turn: an infinite value belongs to the part of
    its own tile alone, and stays infinite (not 0 * inf) where that part has all the weight."""
    a = _Attend("bf16", 4, 4, hd, 16, prefix, [0] * seqs, 2, cuda)  # the first query of each stops a key early
    q = a.q.view(-1, 4, hd)
    q[..., 0] = 8.0
    a.k[..., 0] = 0.0
    tile = key // 128 * 128
    for j in range(tile, min(tile + 128, prefix)):
        a.k[int(a.prefix_table[j // 16]), j % 16, :, 0] = 8.0 * hd ** 0.5   # 64 more than others get
    a.scale *= 4                                                                # 256
    a.v[int(a.prefix_table[key // 16]), key % 16, :, 3] = float("inf")
    for _ in range(10):
        got, _ = a()
        assert (got[..., 3] == np.inf).all() and np.isfinite(np.delete(got, 3, 2)).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,tq", [(1, 1, 1), (4, 2, 8), (4, 2, 20), (2, 2, 65), (8, 1, 40)])
def test_attention_over_an_empty_cache(kind, hq, hkv, tq, cuda):
    """A cache without pages and nothing to see: zero rows, whichever kernel has as many rows."""
    import torch
    import sheaf_b200 as sb

    b, hd = 3, 64
    c = sb.KvCache(None, None, 16 * hkv * hd, hkv * hd, hd, 0, 16, hkv, hd, ELEM[kind])
    q = torch.randn(b * tq, hq * hd, device=cuda).to(torch.float32 if kind == "f32" else torch.bfloat16)
    out, lse = torch.full_like(q, 9.0), torch.full((b * tq, hq), 9.0, device=cuda)
    lens = _i([0, -1, 0], cuda)
    size = sb.lib().sb_op_prefix_attention_workspace_size(c, b, tq, hq, 0, 0)
    ws = torch.full((size // 4 + 4,), float("nan"), device=cuda)
    assert sb.lib().sb_op_prefix_attention(c, q.data_ptr(), hq * hd, out.data_ptr(), hq * hd, lse.data_ptr(), b, tq, hq,
                                           0.125, None, 0, None, 0, lens.data_ptr(), ws.data_ptr(), size,
                                           _stream()) == 0
    assert (out == 0).all() and torch.isneginf(lse).all()


# ---- attention: scores far from zero ----------------------------------------------------


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd,prefix,lens,tq", [(2, 2, 64, 40, [3, 9], 1), (8, 2, 128, 300, [5] * 9, 1),
                                                      (4, 4, 64, 2000, [40] * 80, 1), (2, 1, 128, 0, [300, 5], 40)])
@pytest.mark.parametrize("size", [1e6, 3e9, 1e12, -1e12, 1e30])
def test_attention_of_large_scores(kind, hq, hkv, hd, prefix, lens, tq, size, cuda):
    """Scores of one size (a single product of each query, the same with every key): all visible keys weigh the same,
    or, where a key has none of it, everything or nothing."""
    a = _Attend(kind, hq, hkv, hd, 16, prefix, lens, tq, cuda)
    a.q.zero_()
    a.k.zero_()
    q = a.q.view(-1, hq, hd)
    r = np.arange(1, q.shape[0] * hq + 1).reshape(-1, hq)
    x = np.sqrt(abs(size)) * (1 + (r % 37) / 37)     # of all mantissas
    q[..., 3] = _t(x, kind, cuda) * float(np.sign(size))
    a.k[..., 3] = float(np.sqrt(abs(size)))
    a.scale = 0.7
    odd = np.nonzero(a.lens > 4)[0]
    for s in odd:                                    # the fourth own key of long sequences has a score of 0
        a.k[int(a.table[s][0]), 3, :, 3] = 0.0
    got, lse = a()
    _check_rows(a, got, lse, [(s, t) for s in (0, 1, len(lens) - 1) for t in {0, tq - 1}])
    assert np.isfinite(got).all()


# ---- attention: layouts and kernels side by side ------------------------------------------


@pytest.mark.parametrize("hq,hkv,hd,page,prefix,lens,tq,heads_first,pad", [
    (8, 2, 128, 16, 3000, [100] * 40, 1, True, 8),      # tcgen05: 160 rows, head-major pages
    (4, 4, 64, 24, 1500, [30] * 70, 1, True, 24),       # 70 rows, key tiles dealt out
    (4, 1, 64, 32, 300, [200, 131], 40, True, 8),       # own keys on tcgen05 too
    (4, 1, 32, 128, 300, [200, 131], 40, False, 40),
    (8, 8, 128, 16, 500, [40] * 30, 1, True, 8),        # 4 warps of mma, 128 values a head
    (3, 3, 128, 10, 400, [40] * 50, 1, True, 8),        # pages of 10
    (1, 1, 64, 16, 500, [13000], 40, False, 0),         # 4-warp prefix, tcgen05 own keys beside it
    (1, 1, 128, 16, 13000, [500], 24, True, 8),         # tcgen05 prefix, 4-warp own keys beside it
])
def test_attention_layouts_by_kernel(hq, hkv, hd, page, prefix, lens, tq, heads_first, pad, cuda):
    import torch

    a = _Attend("bf16", hq, hkv, hd, page, prefix, lens, tq, cuda, heads_first=heads_first, pad=pad)
    got, lse = a()
    b = len(lens)
    q, k, v = _f64(a.q), *(_f64(x).swapaxes(1, 2) if heads_first else _f64(x) for x in (a.k, a.v))
    for s, t in {(s, t) for s in (0, b // 2, b - 1) for t in (0, tq // 2, tq - 1)}:
        r = s * tq + t
        one = _attend64(q[r:r + 1, :hq * hd], k, v, a.prefix_table, prefix, a.table[s:s + 1], [lens[s] - tq + t + 1], 1,
                        a.scale, page)
        _check_attention("bf16", got[r:r + 1], lse[r:r + 1], one, hd)
    assert (a.out[:, hq * hd:] == 9).all()
    first = a.out.clone()
    for _ in range(5):
        a()
        assert torch.equal(a.out, first)


# ---- offsets beyond 32 bits, and graphs -----------------------------------------------------


def _far_pages(kind, rows, heads, hd, dev):
    """Nine pages 2^28 elements apart, the last one beyond 2^31, as views of one allocation."""
    import torch

    flat = torch.empty(2 ** 31 + 2 ** 18, device=dev, dtype=torch.float32 if kind == "f32" else torch.bfloat16)
    return flat.as_strided((9, rows, heads, hd), (2 ** 28, heads * hd, hd, 1))


@pytest.mark.parametrize("kind,hq,hkv,hd,prefix,lens,tq", [
    ("bf16", 4, 2, 64, 20, [9, 14], 1),              # a warp
    ("bf16", 8, 1, 128, 30, [9, 14, 16], 3),         # 4 warps
    ("bf16", 8, 1, 128, 64, [40, 64], 40),           # tcgen05
    ("f32", 4, 2, 64, 20, [9, 14], 1),
    ("f32", 8, 1, 128, 30, [9, 14, 16], 3),
])
def test_attention_over_pages_beyond_32_bits(kind, hq, hkv, hd, prefix, lens, tq, cuda):
    a = _Attend(kind, hq, hkv, hd, 64, prefix, lens, tq, cuda)
    want, want_lse = a()
    far = []
    for x in (a.k, a.v):
        y = _far_pages(kind, 64, hkv, hd, cuda)
        y[9 - x.shape[0]:].copy_(x)
        far.append(y)
    shift = 9 - a.k.shape[0]
    a.k, a.v = far
    a.prefix_table, a.table = a.prefix_table + shift, a.table + shift
    got, lse = a()
    assert np.array_equal(got, want) and np.array_equal(lse, want_lse)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_append_beyond_32_bits(kind, cuda):
    import torch
    import sheaf_b200 as sb

    hq, hkv, hd, n, page = 2, 2, 64, 70, 32
    width = (hq + 2 * hkv) * hd
    qkv = torch.randn(n, width, device=cuda).to(torch.float32 if kind == "f32" else torch.bfloat16)
    k, v = (_far_pages(kind, page, hkv, hd, cuda) for _ in range(2))
    pages = [8, 0, 7]
    for x in (k, v):
        x[pages] = 0
    q = torch.zeros(n, hq * hd, device=cuda, dtype=qkv.dtype)
    seq, pos, table = _i(np.zeros(n), cuda), _i(np.arange(n), cuda), _i([pages], cuda)
    assert sb.lib().sb_op_kv_append(_cache((k, v)), qkv.data_ptr(), width, n, hq, q.data_ptr(), hq * hd, seq.data_ptr(),
                                    pos.data_ptr(), 0, table.data_ptr(), 1, 3, 0, 0, None, None, 0, _stream()) == 0
    x = qkv.view(n, hq + 2 * hkv, hd)
    assert torch.equal(q, x[:, :hq].reshape(n, -1))
    for c, part in ((k, x[:, hq:hq + hkv]), (v, x[:, hq + hkv:])):
        assert torch.equal(c[pages].reshape(-1, hkv, hd)[:n], part)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("v", [1000, 9000])
def test_logprobs_of_rows_beyond_32_bits(kind, v, cuda):
    import torch
    import sheaf_b200 as sb

    L, ld, rows, k = sb.lib(), 2 ** 30 + 8, 3, 4
    flat = torch.empty(2 * ld + v, device=cuda, dtype=torch.float32 if kind == "f32" else torch.bfloat16)
    x = flat.as_strided((rows, v), (ld, 1))
    near = torch.randn(rows, v, device=cuda).to(flat.dtype)
    x.copy_(near)
    t, g = _t([5, 0, v - 1], "f32", cuda), _t([1.0, -2.0, 0.5], "f32", cuda)

    def score(p, ld):
        o = torch.zeros(3, rows, device=cuda)
        ids = torch.zeros(rows, k, device=cuda, dtype=torch.int32)
        alt = torch.zeros(rows, k, device=cuda)
        assert L.sb_op_token_logprobs(ELEM[kind], p.data_ptr(), ld, rows, v, t.data_ptr(), 1.0, o[0].data_ptr(),
                                      o[1].data_ptr(), o[2].data_ptr(), k, ids.data_ptr(), alt.data_ptr(),
                                      _stream()) == 0
        return o, ids, alt

    def grad(p, ld, o):
        assert L.sb_op_token_logprobs_bwd(ELEM[kind], p.data_ptr(), ld, rows, v, t.data_ptr(), 1.0, o[2].data_ptr(),
                                          o[1].data_ptr(), g.data_ptr(), g.data_ptr(), p.data_ptr(), ld, _stream()) == 0

    want, got = score(near, v), score(flat, ld)
    assert torch.equal(want[1], got[1])
    assert (want[0] - got[0]).abs().max() < 1e-5 and (want[2] - got[2]).abs().max() < 1e-5
    grad(near, v, want[0])
    grad(flat, ld, want[0])
    assert torch.equal(near, x)


@pytest.mark.parametrize("kind,hq,hkv,hd,prefix,lens,tq", [
    ("bf16", 4, 4, 64, 2000, [40] * 80, 1),     # tcgen05, and a warp's blocks beside it
    ("bf16", 2, 2, 64, 300, [20] * 12, 3),      # 4 warps, and a warp's blocks beside them
    ("bf16", 2, 1, 64, 0, [300, 5], 40),
    ("f32", 4, 2, 64, 300, [5, 60], 2),
])
def test_attention_in_a_graph(kind, hq, hkv, hd, prefix, lens, tq, cuda):
    """Captured once after a first call, replayed with other queries and lengths in the same places."""
    import torch
    import sheaf_b200 as sb

    a = _Attend(kind, hq, hkv, hd, 16, prefix, lens, tq, cuda)
    L, c, b = sb.lib(), _cache((a.k, a.v)), len(lens)
    size = L.sb_op_prefix_attention_workspace_size(c, b, tq, hq, prefix, a.table.shape[1])
    ws = torch.full((size // 4 + 4,), float("nan"), device=cuda)
    pt, t, ln = _i(a.prefix_table, cuda), _i(a.table, cuda), _i(a.lens, cuda)
    q, out = a.q.clone(), torch.zeros_like(a.out)

    def attend():
        assert L.sb_op_prefix_attention(c, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), None, b, tq, hq,
                                        a.scale, pt.data_ptr(), prefix, t.data_ptr(), a.table.shape[1], ln.data_ptr(),
                                        ws.data_ptr(), size, _stream()) == 0

    attend()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            attend()
    for i in range(4):
        a.lens = np.maximum(np.array(lens) - i, 0)
        a.q.mul_(0.75)
        want, _ = a()
        q.copy_(a.q)
        ln.copy_(_i(a.lens, cuda))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(_f64(out).reshape(want.shape), want)
