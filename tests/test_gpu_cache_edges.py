"""Corners of cached generation and scoring: idle slots, NaN and infinities,
logits and scores far from zero, pointers at odd places. Plain restatements
and tolerances as in test_gpu_cache.py."""
import numpy as np
import pytest

from tests.test_gpu_cache import _Attend, _attend64, _check_attention, _f64

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
