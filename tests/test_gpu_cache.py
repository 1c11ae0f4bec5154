"""Appending to a paged cache, attention of sequences that share a prefix in
it, and the scoring of tokens, through the C ABI against plain restatements in
float64 (numpy).

Tolerances follow from the arithmetic. u = 2^-24 and w = 2^-8 are the unit
roundoffs of float32 and bf16 (round to nearest). Outputs that are rounded
once to bf16 lie between the roundings of the float32 bound's ends.
 * rotation: two products and a sum in float32.
 * attention, per output: the probabilities reach the products in the element
   type (bf16: w of sum_j p_j |v_j|), and float32 sums and exponentials leave
   a few u of the same sums; scores are sums of head_dim float32 products,
   whose error moves every probability alike.
 * log probabilities: float32 exponentials and sums of v terms in some order.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ELEM = {"f32": 0x21000020, "bf16": 0x22000010}
U, W = 2.0 ** -24, 2.0 ** -8


def _t(a, kind, dev):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(
        torch.float32 if kind == "f32" else torch.bfloat16).to(dev)


def _i(a, dev):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def _f64(t):
    return t.double().cpu().numpy()


def _stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


def _cache(kv, heads_first=False):
    """The description of k, v [pages, rows, heads, hd], or [pages, heads, rows, hd] with heads_first."""
    import torch
    from sheaf_b200 import KvCache

    k, v = kv
    assert k.stride() == v.stride()
    rows, heads = (2, 1) if heads_first else (1, 2)
    return KvCache(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(rows), k.stride(heads), k.shape[0], k.shape[rows],
                   k.shape[heads], k.shape[3], ELEM["f32" if k.dtype == torch.float32 else "bf16"])


def _within(got, want, bound, kind):
    """Whether `got` is within `bound` of `want`, then rounded to the type."""
    import torch

    low, high = want - bound, want + bound
    if kind == "bf16":
        low, high = (torch.from_numpy(np.ascontiguousarray(a)).to(torch.bfloat16).double().numpy() for a in (low, high))
    return bool(((low <= got) & (got <= high)).all())


def _error():
    import sheaf_b200

    return sheaf_b200.lib().sb_op_device_error()


# ---- append -----------------------------------------------------------------


def _rotate64(x, cos, sin, mode, rot):
    y = x.copy()
    if mode == 1:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    elif mode == 2:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return y


APPEND = [
    # kind, hq, hkv, hd, page, mode, rot, pad (row stride beyond the width), shift (elements off a 16-byte start)
    ("bf16", 6, 6, 64, 16, 0, 0, 0, 0),
    ("bf16", 32, 8, 128, 64, 1, 128, 0, 0),
    ("bf16", 4, 1, 64, 24, 2, 64, 8, 0),
    ("bf16", 3, 1, 32, 5, 1, 16, 8, 0),
    ("bf16", 2, 2, 64, 16, 1, 24, 0, 0),    # half the rotated values is no whole vector
    ("bf16", 2, 1, 64, 16, 2, 64, 1, 0),    # rows that start off 16 bytes
    ("bf16", 2, 1, 64, 16, 1, 64, 0, 3),
    ("f32", 12, 12, 64, 24, 2, 32, 0, 0),
    ("f32", 8, 2, 128, 16, 1, 128, 4, 0),
    ("f32", 1, 1, 32, 1, 1, 2, 1, 1),
    ("f32", 0, 3, 32, 7, 2, 32, 0, 0),      # keys and values alone
]


@pytest.mark.parametrize("kind,hq,hkv,hd,page,mode,rot,pad,shift", APPEND)
def test_append(kind, hq, hkv, hd, page, mode, rot, pad, shift, cuda):
    import torch
    import sheaf_b200 as sb

    rng = np.random.default_rng(hd + rot + hq)
    n_seqs, max_pages, base = 3, 4, 11
    width = (hq + 2 * hkv) * hd
    # ragged: sequence 0 gets a run that crosses a page, 1 one token, 2 its last place; and a padding token
    seq = np.array([0] * min(4, page * 2) + [1, -1, 2])
    pos = base + np.array(list(range(page - 1, page - 1 + min(4, page * 2))) + [0, 0, page * max_pages - 1])
    n = len(seq)
    n_pos = base + page * max_pages
    flat = torch.zeros(n * (width + pad) + shift + 16, device=cuda,
                       dtype=torch.float32 if kind == "f32" else torch.bfloat16)
    qkv = flat[shift:shift + n * (width + pad)].view(n, width + pad)
    qkv.copy_(_t(rng.standard_normal((n, width + pad)), kind, cuda))
    k, v = (_t(rng.standard_normal((n_seqs * max_pages + 1, page, hkv, hd)), kind, cuda) for _ in range(2))
    k0, v0 = _f64(k), _f64(v)
    table = rng.permutation(n_seqs * max_pages + 1)[:n_seqs * max_pages].reshape(n_seqs, max_pages)
    ang = np.arange(n_pos)[:, None] * 100.0 ** (-np.arange(max(rot, 2) // 2) / max(rot, 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    q_out = torch.full((n, max(hq, 1) * hd), 7.0, device=cuda, dtype=qkv.dtype)
    seq_d, pos_d, table_d, cos_d, sin_d = _i(seq, cuda), _i(pos, cuda), _i(table, cuda), _t(cos, "f32", cuda), \
        _t(sin, "f32", cuda)
    c = _cache((k, v))
    rc = sb.lib().sb_op_kv_append(c, qkv.data_ptr(), width + pad, n, hq, q_out.data_ptr() if hq else None,
                                  q_out.stride(0), seq_d.data_ptr(), pos_d.data_ptr(), base, table_d.data_ptr(), n_seqs,
                                  max_pages, mode, rot, cos_d.data_ptr(), sin_d.data_ptr(), n_pos, _stream())
    assert rc == 0 and _error() == 0
    x = _f64(qkv)[:, :width].reshape(n, hq + 2 * hkv, hd)
    cs, sn = cos.astype(np.float64)[pos][:, None], sin.astype(np.float64)[pos][:, None]
    turned = _rotate64(x[:, :hq + hkv], cs, sn, mode, rot)
    turned[seq < 0] = 0
    for i in np.nonzero(seq >= 0)[0]:
        own = pos[i] - base
        p = table[seq[i], own // page], own % page
        k0[p], v0[p] = turned[i, hq:], x[i, hq + hkv:]
    # a product's error is u of it, the sum's u of the sum
    amp = 2 * np.abs(x).max() * 3 * U
    assert np.array_equal(_f64(v), v0)
    assert _within(_f64(k), k0, amp, kind)
    if hq:
        assert _within(_f64(q_out).reshape(n, hq, hd), turned[:, :hq], amp, kind)
        assert (q_out[seq_d < 0] == 0).all()
    if mode == 0:
        assert np.array_equal(_f64(k), k0)


def test_append_in_place_and_outside_its_tables(cuda):
    """q_out may be qkv itself; positions, sequences and pages outside their tables are skipped and reported."""
    import torch
    import sheaf_b200 as sb

    L = sb.lib()
    rng = np.random.default_rng(3)
    hq, hkv, hd, page = 4, 2, 64, 8
    width = (hq + 2 * hkv) * hd
    qkv = _t(rng.standard_normal((5, width)), "bf16", cuda)
    before = qkv.clone()
    k, v = (torch.zeros(4, page, hkv, hd, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    cos, sin = torch.zeros(64, 32, device=cuda), torch.ones(64, 32, device=cuda)  # a quarter turn
    table = _i([[0, 1], [99, 3]], cuda)

    def append(seq, pos):
        seq, pos = _i(seq, cuda), _i(pos, cuda)
        return L.sb_op_kv_append(_cache((k, v)), qkv.data_ptr(), width, 5, hq, qkv.data_ptr(), width,
                                 seq.data_ptr(), pos.data_ptr(), 0, table.data_ptr(), 2, 2, 1, 64,
                                 cos.data_ptr(), sin.data_ptr(), 64, _stream())

    assert append([0, 0, 0, 1, 1], [0, 1, 9, 8, 15]) == 0 and _error() == 0
    q = before.view(5, hq + 2 * hkv, hd)[:, :hq + hkv]
    want = torch.cat([-q[..., 32:], q[..., :32]], -1)
    assert torch.equal(qkv.view(5, -1, hd)[:, :hq], want[:, :hq])
    assert torch.equal(qkv.view(5, -1, hd)[:, hq:], before.view(5, -1, hd)[:, hq:])
    assert torch.equal(k[[0, 0, 1, 3, 3], [0, 1, 1, 0, 7]], want[:, hq:])
    kept = k.clone()
    qkv.copy_(before)
    # a sequence past the table, a position past its pages, one below 0, a page outside the cache, padding
    assert append([2, 0, 0, 1, -1], [0, 16, -1, 0, 0]) == 0
    assert _error() == 2 and _error() == 0
    assert torch.equal(k, kept)
    assert (qkv[[0, 1, 2, 4], :hq * hd] == 0).all()
    assert torch.equal(qkv.view(5, -1, hd)[3, :hq], want[3, :hq])


# ---- attention --------------------------------------------------------------


def _attend64(q, k, v, prefix_table, prefix, table, lens, tq, scale, page):
    """out, lse, sum_j p_j |v_j| and max_j sum_c |q_c k_c| scale, in float64. k, v [pages, rows, heads, hd]."""
    b, (hkv, hd) = len(lens), k.shape[2:]
    hq = q.shape[1] // hd
    g = hq // hkv
    out, amp = np.zeros((b * tq, hq, hd)), np.zeros((b * tq, hq, hd))
    lse, score = np.full((b * tq, hq), -np.inf), np.zeros((b * tq, hq))
    shared = [(prefix_table[j // page], j % page) for j in range(prefix)]
    for s in range(b):
        if lens[s] < 0:
            continue
        at = shared + [(table[s][j // page], j % page) for j in range(lens[s])]
        if not at:
            continue
        pg, rw = np.array(at).T
        ks, vs = k[pg, rw], v[pg, rw]
        for t in range(tq):
            n = prefix + lens[s] - tq + t + 1
            if n <= 0:
                continue
            for h in range(hq):
                x = q[s * tq + t].reshape(hq, hd)[h]
                z = ks[:n, h // g] @ x * scale
                m = z.max()
                p = np.exp(z - m)
                o = s * tq + t, h
                with np.errstate(invalid="ignore"):
                    out[o] = p @ vs[:n, h // g] / p.sum()
                    amp[o] = p @ np.abs(vs[:n, h // g]) / p.sum()
                lse[o] = m + np.log(p.sum())
                score[o] = (np.abs(ks[:n, h // g]) @ np.abs(x)).max() * scale
    return out, lse, amp, score


def _check_attention(kind, got, got_lse, want, hd):
    out, lse, amp, score = want
    # every probability carries the errors of its score (hd products) and exponential, and the type's rounding
    rel = 2 * (hd + 8) * U * np.maximum(score, 1.0)[..., None] + (W if kind == "bf16" else 64 * U)
    bound = rel * amp + 1e-30
    assert np.array_equal(np.isnan(got), np.isnan(out))
    ok = ~np.isnan(out)
    assert _within(got[ok], out[ok], bound[ok], kind), float((np.abs(got - out)[ok] / bound[ok]).max())
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got_lse), empty) and (got[empty] == 0).all()
    b = (2 * (hd + 8) * U * np.maximum(score, 1.0) + 64 * U * np.maximum(np.abs(lse), 1))[~empty]
    assert (np.abs(got_lse - lse)[~empty] <= b).all()


class _Attend:
    """A random cache, page tables, queries and lengths, and a call on them."""

    def __init__(self, kind, hq, hkv, hd, page, prefix, lens, tq, dev, seed=0, heads_first=False, pad=0, capacity=None):
        import torch

        rng = np.random.default_rng(seed + hd + page + prefix)
        self.kind, self.hq, self.hd, self.page, self.prefix, self.tq, self.dev = kind, hq, hd, page, prefix, tq, dev
        self.lens, b = np.array(lens), len(lens)
        per = -(-max(max(lens), 0 if capacity is None else capacity) // page)
        n_prefix = -(-prefix // page)
        n = max(1, b * per + n_prefix)
        order = rng.permutation(n)
        self.prefix_table, self.table = order[:n_prefix], order[n_prefix:n_prefix + b * per].reshape(b, per)
        shape = (n, hkv, page, hd) if heads_first else (n, page, hkv, hd)
        self.k, self.v = (_t(rng.standard_normal(shape), kind, dev) for _ in range(2))
        self.heads_first = heads_first
        self.q = torch.zeros(b * tq, hq * hd + pad, device=dev, dtype=self.k.dtype)
        self.q[:, :hq * hd] = _t(rng.standard_normal((b * tq, hq * hd)) * 2, kind, dev)
        self.out = torch.full((b * tq, hq * hd + pad), 9.0, device=dev, dtype=self.k.dtype)
        self.lse = torch.full((b * tq, hq), 9.0, device=dev)
        self.scale = 1 / math.sqrt(hd)

    def __call__(self, lse=True):
        import torch
        import sheaf_b200 as sb

        L = sb.lib()
        c = _cache((self.k, self.v), self.heads_first)
        b = len(self.lens)
        size = L.sb_op_prefix_attention_workspace_size(c, b, self.tq, self.hq, self.prefix, self.table.shape[1])
        # NaN everywhere: a partial result that nothing wrote must not be read
        ws = torch.full((size // 4 + 4,), float("nan"), device=self.dev)
        pt, t, ln = _i(self.prefix_table, self.dev), _i(self.table, self.dev), _i(self.lens, self.dev)
        rc = L.sb_op_prefix_attention(c, self.q.data_ptr(), self.q.stride(0), self.out.data_ptr(), self.out.stride(0),
                                      self.lse.data_ptr() if lse else None, b, self.tq, self.hq, self.scale,
                                      pt.data_ptr(), self.prefix, t.data_ptr(), self.table.shape[1], ln.data_ptr(),
                                      ws.data_ptr(), size, _stream())
        assert rc == 0
        torch.cuda.synchronize()
        n = self.hq * self.hd
        return _f64(self.out)[:, :n].reshape(-1, self.hq, self.hd), _f64(self.lse)

    def want(self):
        k, v = _f64(self.k), _f64(self.v)
        if self.heads_first:
            k, v = k.swapaxes(1, 2), v.swapaxes(1, 2)
        return _attend64(_f64(self.q)[:, :self.hq * self.hd], k, v, self.prefix_table, self.prefix, self.table,
                         self.lens, self.tq, self.scale, self.page)

    def check(self):
        got, lse = self()
        _check_attention(self.kind, got, lse, self.want(), self.hd)


ATTEND = [
    # hq, hkv, hd, page, prefix, lens, tq
    (6, 6, 64, 16, 200, [1, 33, 0, 56], 1),
    (8, 2, 128, 16, 300, [5, -1, 64, 1], 1),
    (32, 8, 32, 24, 129, [40], 1),
    (8, 1, 64, 7, 0, [1, 65, 20], 1),            # no prefix: one token up to more than a tile, odd pages
    (4, 4, 64, 16, 100, [0, 0], 1),              # nothing but the prefix
    (2, 1, 128, 64, 1, [1], 1),
    (12, 12, 64, 24, 77, [37, 40, 55], 37),      # many new tokens a sequence: a causal edge inside tiles
    (4, 2, 64, 16, 50, [3, 8, 1, -1], 5),        # more queries than keys: some see the prefix alone
    (4, 2, 32, 16, 0, [3, 130], 5),              # or nothing
    (4, 1, 128, 32, 260, [70, 66], 66),
    (64, 1, 64, 16, 130, [9, 17], 2),            # 64 query heads on one key head
    (2, 2, 64, 16, 20, [2] * 70, 1),             # many sequences
    (16, 2, 128, 128, 1030, [129] * 9, 2),
]


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,hd,page,prefix,lens,tq", ATTEND)
def test_attention(kind, hq, hkv, hd, page, prefix, lens, tq, cuda):
    _Attend(kind, hq, hkv, hd, page, prefix, lens, tq, cuda).check()
    assert _error() == 0


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_strides(kind, cuda):
    """Head-major pages, rows of q and out further apart, no lse."""
    a = _Attend(kind, 8, 4, 64, 16, 90, [17, 4, 30], 3, cuda, heads_first=True, pad=8)
    a.check()
    assert (a.out[:, a.hq * a.hd:] == 9).all()
    first = a.out.clone()
    a.out.fill_(9.0)
    a(lse=False)
    assert bool((a.out == first).all())


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("prefix,lens,tq", [(8200, [100] * 40, 1), (3000, [300, 200], 70), (20000, [3], 1)])
def test_attention_longer(kind, prefix, lens, tq, cuda):
    """Keys cut over many blocks. Sampled rows against float64."""
    a = _Attend(kind, 8, 2, 128, 16, prefix, lens, tq, cuda)
    got, lse = a()
    rows = sorted({0, len(lens) * tq - 1, (len(lens) // 2) * tq})
    for r in rows:
        s, t = divmod(r, tq)
        one = _attend64(_f64(a.q)[r:r + 1], _f64(a.k), _f64(a.v), a.prefix_table, prefix, a.table[s:s + 1],
                        [lens[s] - tq + t + 1], 1, a.scale, a.page)
        _check_attention(kind, got[r:r + 1], lse[r:r + 1], one, 128)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_repeats_bit_for_bit_on_any_stream(kind, cuda):
    import torch

    a = _Attend(kind, 8, 2, 64, 16, 900, [100, 3, 77], 2, cuda)
    a()
    first, first_lse = a.out.clone(), a.lse.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a.out.zero_()
        a()
    side.synchronize()
    assert torch.equal(a.out, first) and torch.equal(a.lse, first_lse)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_keeps_unseen_keys_out(kind, cuda):
    """NaN and infinities in rows of the cache that no query sees: past a sequence's end, in unused pages, past the
    prefix's end; and in a key that only later queries see."""
    a = _Attend(kind, 4, 2, 64, 16, 40, [20, 3], 2, cuda, capacity=48)
    clean, _ = a()
    pg = a.prefix_table[2]
    for x in (a.k, a.v):
        x[int(pg), 8:] = float("nan")                   # prefix: 40 = 2 pages and 8 rows
        x[int(a.table[0][1]), 4:] = float("inf")        # sequence 0: 20 = 1 page and 4 rows
        x[int(a.table[1][0]), 3:] = float("nan")
        x[int(a.table[1][2])] = float("-inf")
    got, _ = a()
    assert np.array_equal(got, clean)
    a.v[int(a.table[0][1]), 3, :, 5] = float("nan")     # the last token's values: its own query alone sees them
    got, lse = a()
    assert np.array_equal(got[0], clean[0]) and np.array_equal(got[2:], clean[2:])
    assert np.isnan(got[1][:, 5]).all() and np.array_equal(np.delete(got[1], 5, 1), np.delete(clean[1], 5, 1))


def test_attention_calls_in_a_row(cuda):
    """Calls whose kernels overlap, one after the other in one workspace, without a wait between them."""
    import torch
    import sheaf_b200 as sb

    a = _Attend("bf16", 32, 8, 64, 16, 4096, [100] * 40, 1, cuda)
    L, c, b = sb.lib(), _cache((a.k, a.v)), len(a.lens)
    size = L.sb_op_prefix_attention_workspace_size(c, b, 1, a.hq, a.prefix, a.table.shape[1])
    ws = torch.empty(size // 4 + 4, device=cuda)
    pt, t, ln = _i(a.prefix_table, cuda), _i(a.table, cuda), _i(a.lens, cuda)
    qs = [a.q * (1 - i / 8) for i in range(8)]
    outs = [torch.empty_like(a.out) for _ in range(16)]

    def attend(q, out):
        assert L.sb_op_prefix_attention(c, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), None, b, 1, a.hq,
                                        a.scale, pt.data_ptr(), a.prefix, t.data_ptr(), a.table.shape[1],
                                        ln.data_ptr(), ws.data_ptr(), size, _stream()) == 0

    for q, out in zip(qs, outs[:8]):
        attend(q, out)
        torch.cuda.synchronize()
    for _ in range(20):
        for out in outs[8:]:
            out.zero_()
        for q, out in zip(qs, outs[8:]):
            attend(q, out)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs[:8], outs[8:]))


@pytest.mark.parametrize("kind,seqs,prefix", [("bf16", 3, 20000), ("bf16", 20, 1500), ("bf16", 70, 20000),
                                              ("f32", 3, 20000), ("f32", 70, 20000)])
def test_attention_keys_at_minus_infinity(kind, seqs, prefix, cuda):
    """Seen keys with a score of -inf weigh nothing, however many come first and however low the others' scores."""
    a = _Attend(kind, 8, 8, 32, 16, prefix, [5] * seqs, 1, cuda)
    q = a.q.view(-1, 8, 32)
    q[..., 0], q[..., 1] = 1.0, 32.0
    a.k[..., 1] = -100.0
    closed = np.arange(len(a.prefix_table)) % 32 < 20   # 320 keys of every 512
    closed[-1] = False
    a.k[_i(a.prefix_table[closed], cuda).long(), ..., 0] = float("-inf")
    got, lse = a()
    for r in (0, seqs // 2, seqs - 1):
        open_ = a.prefix_table[~closed]
        one = _attend64(_f64(a.q)[r:r + 1], _f64(a.k), _f64(a.v), open_, a.prefix - 16 * int(closed.sum()),
                        a.table[r:r + 1], [5], 1, a.scale, 16)
        _check_attention(kind, got[r:r + 1], lse[r:r + 1], one, 32)


def test_attention_reports_indices_outside(cuda):
    a = _Attend("bf16", 4, 2, 64, 16, 40, [20, 16], 1, cuda)
    a.lens = np.array([20, 33])  # two pages hold 32
    got, _ = a()
    assert _error() == 2
    a.lens = np.array([20, 32])
    want, _ = a()
    assert np.array_equal(got, want) and _error() == 0
    a.table[1][0] = 10 ** 6
    a()
    assert _error() == 2


# ---- log probabilities ------------------------------------------------------


def _score64(x, t, temperature):
    z = x / temperature
    m = z.max(1, keepdims=True)
    m = np.where(np.isneginf(m), 0, m)
    with np.errstate(divide="ignore", invalid="ignore"):
        log_sum = np.log(np.exp(z - m).sum(1, keepdims=True))
        lse = m + log_sum
        lse = np.where(lse < -np.finfo(np.float32).max, -np.inf, lse)  # -inf where float32 cannot hold it
        lp = np.where(np.isneginf(z), -np.inf, (z - m) - log_sum)  # m + log_sum may have lost log_sum
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * lp, 0).sum(1)
    known = (t == np.floor(t)) & (t >= 0) & (t < x.shape[1])
    at = np.where(known, t, 0).astype(int)
    logp = np.where(known, lp[np.arange(len(t)), at], 0.0)
    return lp, p, lse[:, 0], entropy, logp, known, at


def _logits(rows, v, seed, kind):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, v)) * 3
    x[::3] = np.round(x[::3])                        # many equal logits
    if rows > 4:
        x[1] = 2.5                                   # all equal
        x[2] = np.sort(x[2])                         # rising: a thread holds neighbours of the best
        x[3] = -x[2]
        x[4, v // 2] += 60                           # one sure token
    if rows > 8:
        x[5, : v // 2] = -np.inf
        x[6, :] = -np.inf                            # nothing left
        x[7, 1:] = -np.inf                           # one left
        x[8] = -3.3e38                               # the type's lowest values
    import torch

    y = torch.from_numpy(x.astype(np.float32))
    y = y if kind == "f32" else y.to(torch.bfloat16)
    return y


def _best(x, k):
    """Larger first, NaN before all, then the lower index."""
    key = np.where(np.isnan(x), np.inf, x)
    return np.array([sorted(range(x.shape[1]), key=lambda j: (not np.isnan(r[j]), -kk[j], j))[:k]
                     for r, kk in zip(x, key)])


SCORE = [(3, 1, 1), (12, 2, 2), (12, 33, 32), (12, 65, 20), (12, 1000, 8), (12, 1031, 32), (9, 2051, 5),
         (12, 5000, 32), (12, 9001, 1), (4, 50304, 5), (12, 50257, 20), (2, 131072, 8), (300, 6000, 8)]


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,v,k", SCORE)
@pytest.mark.parametrize("pad,temperature", [(0, 1.0), (3, 0.7)])
def test_logprobs(kind, rows, v, k, pad, temperature, cuda):
    import torch
    import sheaf_b200 as sb

    x = _logits(rows, v, rows + v, kind)
    buf = torch.zeros(rows, v + pad, dtype=x.dtype, device=cuda)
    buf[:, :v] = x.to(cuda)
    buf[:, v:] = 1e6  # beyond the row
    x64 = x.double().numpy()
    rng = np.random.default_rng(v)
    t = rng.integers(0, v, rows).astype(np.float32)
    t[: min(3, rows)] = [v, -1, 0.5][: min(3, rows)]
    td = torch.from_numpy(t).to(cuda)
    f = dict(device=cuda, dtype=torch.float32)
    logp, ent, lse, alt = (torch.full(s, 9.0, **f) for s in ((rows,), (rows,), (rows,), (rows, k)))
    ids = torch.full((rows, k), -9, device=cuda, dtype=torch.int32)
    rc = sb.lib().sb_op_token_logprobs(ELEM[kind], buf.data_ptr(), v + pad, rows, v, td.data_ptr(), temperature,
                                       logp.data_ptr(), ent.data_ptr(), lse.data_ptr(), k, ids.data_ptr(),
                                       alt.data_ptr(), _stream())
    assert rc == 0
    lp, p, lse64, ent64, logp64, known, at = _score64(x64, t.astype(np.float64), np.float32(temperature).astype(np.float64))
    ids64 = _best(x64, k)
    assert np.array_equal(ids.cpu().numpy(), ids64)
    # log2 units: y = (x - m) c is rounded twice, the exponential has 2^-22, and sums of v terms stay under
    # 64 roundings (pairwise over threads); lse also carries the rounding of m / T
    spread = np.where(np.isfinite(x64), x64, np.nan)
    with np.errstate(all="ignore"):
        import warnings
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            m = np.nanmax(spread, 1) / temperature
    m = np.nan_to_num(m)
    for got, want, size in ((lse, lse64, np.abs(m)), (logp, logp64, np.zeros(rows))):
        got = _f64(got)
        assert np.array_equal(np.isneginf(got), np.isneginf(want))
        ok = np.isfinite(want)
        err = np.abs(got[ok] - want[ok])
        assert (err <= 1e-6 + 256 * U * np.abs(want[ok]).clip(0, 1) + 4 * U * (np.abs(want[ok]) + size[ok])).all(), err.max()
    assert (np.abs(_f64(ent) - ent64) <= 256 * U * np.maximum(ent64, 0.05)).all()
    a64 = np.take_along_axis(lp, ids64, 1)
    a = _f64(alt)
    assert np.array_equal(np.isneginf(a), np.isneginf(a64))
    ok = np.isfinite(a64)
    assert (np.abs(a - a64)[ok] <= 1e-6 + 16 * U * (1 + np.abs(a64[ok]))).all()


@pytest.mark.parametrize("v", [40, 700, 5000, 60000])
def test_logprobs_nan_and_inf(v, cuda):
    import torch
    import sheaf_b200 as sb

    x = np.random.default_rng(v).standard_normal((4, v)).astype(np.float32)
    x[0, [0, v - 1]] = np.nan
    x[1, v // 2] = np.inf
    x[2] = np.nan
    xd = torch.from_numpy(x).to(cuda)
    o = torch.zeros(3, 4, device=cuda)
    ids = torch.zeros(4, 6, device=cuda, dtype=torch.int32)
    alt = torch.zeros(4, 6, device=cuda)
    t = torch.zeros(4, device=cuda)
    assert sb.lib().sb_op_token_logprobs(ELEM["f32"], xd.data_ptr(), v, 4, v, t.data_ptr(), 1.0, o[0].data_ptr(),
                                         o[1].data_ptr(), o[2].data_ptr(), 6, ids.data_ptr(), alt.data_ptr(),
                                         _stream()) == 0
    assert torch.isnan(o[:, :3]).all() and torch.isfinite(o[:, 3]).all() and torch.isnan(alt[:3]).all()
    assert np.array_equal(ids.cpu().numpy(), _best(x, 6))


def test_logprobs_outputs_are_optional(cuda):
    import torch
    import sheaf_b200 as sb

    x = torch.randn(5, 3000, device=cuda)
    lse = torch.zeros(5, device=cuda)
    assert sb.lib().sb_op_token_logprobs(ELEM["f32"], x.data_ptr(), 3000, 5, 3000, None, 1.0, None, None,
                                         lse.data_ptr(), 4, None, None, _stream()) == 0
    torch.cuda.synchronize()
    assert (lse - torch.logsumexp(x, 1)).abs().max() < 1e-5


def _vjp(kind, x, t, temperature, lse, ent, dlogp, dent, dev, in_place=False, pad=0):
    import torch
    import sheaf_b200 as sb

    rows, v = x.shape
    buf = torch.zeros(rows, v + pad, dtype=x.dtype, device=dev)
    buf[:, :v] = x.to(dev)
    dx = buf if in_place else torch.full((rows, v + pad + 1), 7.0, dtype=x.dtype, device=dev)
    f = [torch.from_numpy(np.asarray(a, np.float32)).to(dev) if a is not None else None
         for a in (t, lse, ent, dlogp, dent)]
    p = [a.data_ptr() if a is not None else None for a in f]
    assert sb.lib().sb_op_token_logprobs_bwd(ELEM[kind], buf.data_ptr(), v + pad, rows, v, p[0], temperature, p[1],
                                             p[2], p[3], p[4], dx.data_ptr(), dx.stride(0), _stream()) == 0
    torch.cuda.synchronize()
    if not in_place:
        assert (dx[:, v:] == 7).all()
    return _f64(dx[:, :v])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,v", [(3, 1), (12, 33), (12, 65), (12, 1031), (10, 9001), (9, 50304)])
@pytest.mark.parametrize("in_place,pad,temperature", [(False, 0, 1.0), (True, 0, 0.7), (False, 5, 1.3)])
def test_logprobs_vjp(kind, rows, v, in_place, pad, temperature, cuda):
    x = _logits(rows, v, rows + v, kind)
    x64 = x.double().numpy()
    rng = np.random.default_rng(v + 1)
    t = rng.integers(0, v, rows).astype(np.float32)
    t[: min(3, rows)] = [v, -1, 0.5][: min(3, rows)]
    T = float(np.float32(temperature))
    lp, p, lse, ent, _, known, at = _score64(x64, t.astype(np.float64), T)
    lse32, ent32 = lse.astype(np.float32), ent.astype(np.float32)
    g, h = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    one = np.zeros((rows, v))
    one[np.nonzero(known)[0], at[known]] = 1
    for dlogp, dent in ((g, h), (g, None), (None, h)):
        gg = np.zeros((rows, 1)) if dlogp is None else (g * known)[:, None].astype(np.float64)
        hh = np.zeros((rows, 1)) if dent is None else h[:, None].astype(np.float64)
        plp = np.where(p > 0, p * np.where(p > 0, lp, 0), 0)
        want = (gg * (one - p) - hh * (plp + p * ent[:, None])) / T
        want[np.isneginf(lse32)] = 0  # as defined for a row whose lse is -inf
        got = _vjp(kind, x, t if dlogp is not None else None, temperature, lse32, ent32 if dent is not None else None,
                   dlogp, dent, cuda, in_place, pad)
        # p carries the errors of x / T - lse: the rounding of lse and of x / T, both up to max |x - lse| u
        big = np.where(np.isfinite(x64) & (p > 1e-30), np.abs(x64), 0).max(1, keepdims=True) / T
        size = np.where(np.isfinite(lse), np.abs(lse), 0)[:, None] + big + 8
        terms = (np.abs(gg) * (one + p) + np.abs(hh) * (np.abs(plp) + p * ent[:, None] + p)) / T
        bound = 8 * U * size * terms + 1e-37
        assert _within(got, want, bound, kind), (np.abs(got - want) / bound).max()


def test_logprobs_vjp_against_differences(cuda):
    """sum g logp + h H of the forward entry point, by central differences of single float32 logits."""
    import torch
    import sheaf_b200 as sb

    L = sb.lib()
    rng = np.random.default_rng(8)
    rows, v, T = 6, 37, 0.9
    x = rng.standard_normal((rows, v)).astype(np.float32)
    t = rng.integers(0, v, rows).astype(np.float32)
    g, h = rng.standard_normal(rows), rng.standard_normal(rows)

    def loss(a):
        ad, td = torch.from_numpy(a).to(cuda), torch.from_numpy(t).to(cuda)
        o = torch.zeros(3, rows, device=cuda)
        assert L.sb_op_token_logprobs(ELEM["f32"], ad.data_ptr(), v, rows, v, td.data_ptr(), T, o[0].data_ptr(),
                                      o[1].data_ptr(), o[2].data_ptr(), 0, None, None, _stream()) == 0
        lp, e, l = _f64(o)
        return g * lp + h * e, l, e

    _, lse, ent = loss(x)
    got = _vjp("f32", torch.from_numpy(x), t, T, lse, ent, g, h, cuda)
    step = 2.0 ** -5
    for j in range(0, v, 5):
        up, down = x.copy(), x.copy()
        up[:, j] += step
        down[:, j] -= step
        diff = (loss(up)[0] - loss(down)[0]) / (up[:, j] - down[:, j]).astype(np.float64)
        # truncation: step^2 / 6 times a third derivative of a few |g| + |h|; rounding: 1e-6 over a step
        assert (np.abs(diff - got[:, j]) <= (np.abs(g) + 4 * np.abs(h)) * (2 * step ** 2 + 1e-6 / step)).all()
