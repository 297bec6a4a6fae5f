"""Infinities that a row sees come out of ``Attention`` as the formulas have them: an infinity in a value is one in the result, a
key whose score is minus infinity counts as none, and what is minus infinity plus infinity is NaN.  Tolerances: attention_oracle."""
import numpy as np
import pytest

import attention_oracle as ao
from test_gpu_attention import Problem, check
from test_gpu_join import Array

pytestmark = pytest.mark.gpu
INF = np.inf
# one or few workgroups of a tile a wave, many of common tiles; f32 rows of 128 have the latter alone
SHAPES = [((4, 2, 64), 1), ((2, 2, 128), 1), ((16, 8, 64), 40), ((3, 3, 40), 1), ((16, 16, 104), 40)]


def replace(p, name, value):
    setattr(p, "d" + name, Array(p.dev, value.shape, p.dtype, value))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,copies", SHAPES)
def test_infinite_values(device, dtype, heads, copies):
    n = 150
    p = Problem(device, [n] * copies, 0, heads, dtype, backward=False)
    want = p.wanted(backward=False)
    first, group = (copies - 1) * n, heads[0] // heads[1]  # of the last sequence
    v = p.v.copy()
    # column 5: infinity from row 20 on; 6: minus infinity from row 100 on; 7: both from row 75 on
    v[first + 20, 0, 5], v[first + 100, 0, 6], v[first + 70, 0, 7], v[first + 75, 0, 7] = INF, -INF, INF, -INF
    replace(p, "v", v)
    got = p.forward()
    for col, row, value in ((5, 20, INF), (6, 100, -INF), (7, 70, INF)):
        rows = got["out"][first + row:first + (75 if col == 7 else n), :group, col]
        assert (rows == value).all(), (col, rows[rows != value][:4])
    assert np.isnan(got["out"][first + 75:, :group, 7]).all()
    bad = ~np.isfinite(got["out"])
    assert bad.sum() == group * (130 + 50 + 80)
    check({"out": np.where(bad, 0, got["out"]), "lse": got["lse"]},
          {"out": (np.where(bad, 0, want["out"][0]), want["out"][1]), "lse": want["lse"]}, dtype)
    p.op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,copies", SHAPES)
def test_infinite_scores(device, dtype, heads, copies):
    """A key of minus infinity in one column: rows with a positive number there see it as masked, the others' sums are NaN."""
    n, at = 150, 70
    p = Problem(device, [n] * copies, 0, heads, dtype, backward=False)
    first, group = (copies - 1) * n, heads[0] // heads[1]
    k = p.k.copy()
    k[first + at, 0, 1] = -INF
    replace(p, "k", k)
    got = p.forward()
    seen = ao.seen(n, n, True)
    for h in range(group):
        q, k, v = (a[first:first + n, i].astype(np.float64) for a, i in ((p.q, h), (p.k, 0), (p.v, 0)))
        assert (q[at:, 1] != 0).all()
        mask = seen.copy()
        mask[:, at] = False  # (of the rows that are checked)
        want = ao.head(q, k, v, mask, p.scale, dtype)
        spoilt = (np.arange(n) >= at) & (q[:, 1] < 0)
        assert spoilt.any() and not spoilt[at:].all()
        assert np.isnan(got["out"][first:first + n, h][spoilt]).all() and np.isnan(got["lse"][h, first:first + n][spoilt]).all()
        out, lse = got["out"][first:first + n, h][~spoilt], got["lse"][h, first:first + n][~spoilt]
        assert (np.abs(out - want["out"][0][~spoilt]) <= want["out"][1][~spoilt]).all(), h
        assert (np.abs(lse - want["lse"][0][~spoilt]) <= want["lse"][1][~spoilt]).all(), h
    p.op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,copies", SHAPES)
def test_infinite_gradients(device, dtype, heads, copies):
    """An infinity in a row's gradient: the values that this row sees get it, what the row has no part in comes out as without it."""
    n, at = 150, 70
    p = Problem(device, [n] * copies, 0, heads, dtype)
    want = p.wanted()
    first, group = (copies - 1) * n, heads[0] // heads[1]
    p.forward()
    go = p.go.copy()
    go[first + at, 0, 2] = -INF
    replace(p, "go", go)
    got = p.backward()
    assert (got["grad_v"][first:first + at + 1, 0, 2] == -INF).all()
    clean = {name: np.ones(a.shape, bool) for name, a in got.items()}
    clean["grad_q"][first + at, 0] = False
    clean["grad_k"][first:first + at + 1, 0] = False
    clean["grad_v"][first:first + at + 1, 0, 2] = False
    assert not np.isfinite(got["grad_q"][first + at, 0]).any() and not np.isfinite(got["grad_k"][first:first + at + 1, 0]).any()
    check({name: np.where(c, got[name], 0) for name, c in clean.items()},
          {name: (np.where(c, want[name][0], 0), want[name][1]) for name, c in clean.items()}, dtype)
    assert group >= 1
    p.op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,copies", [((4, 2, 64), 1), ((8, 8, 104), 40)])
def test_rows_side_by_side_off_their_boundaries(device, dtype, heads, copies):
    """q, k and v in one array that starts three elements off, rows of nothing between the sequences."""
    n = 140
    p = Problem(device, [n] * copies, 0, heads, dtype, gap=2, shift=3, fused=True)
    want = p.wanted()
    first, group = p.begin[-1], heads[0] // heads[1]
    at = (p.h + p.kv) * p.d + 5  # column 5 of kv head 0's values
    both = np.concatenate([a.reshape(p.rows, -1) for a in (p.q, p.k, p.v)] + [np.full((p.rows, 8), np.nan, np.float32)], axis=1)
    clean = p.all
    both[first + 90, at], both[first + 91, at + 1] = -INF, INF
    p.all = Array(device, both.shape, dtype, both, 3)
    got = p.forward()
    bad = ~np.isfinite(got["out"]) & ~np.isnan(want["out"][0])
    assert (got["out"][first + 90:first + n, :group, 5] == -INF).all() and (got["out"][first + 91:first + n, :group, 6] == INF).all()
    assert bad.sum() == group * (50 + 49)
    check({"out": np.where(bad, 0, got["out"]), "lse": got["lse"]}, {"out": (np.where(bad, 0, want["out"][0]), want["out"][1]), "lse": want["lse"]}, dtype)
    p.all = clean
    p.forward()
    go = p.go.copy()
    go[first + 90, 0, 2] = INF
    p.dgo = Array(device, go.shape, dtype, go, 3)
    got = p.backward()
    assert (got["grad_v"][first:first + 91, 0, 2] == INF).all()
    spoilt = {name: np.zeros(a.shape, bool) for name, a in got.items()}
    spoilt["grad_q"][first + 90, 0] = spoilt["grad_k"][first:first + 91, 0] = spoilt["grad_v"][first:first + 91, 0, 2] = True
    check({name: np.where(s, 0, got[name]) for name, s in spoilt.items()},
          {name: (np.where(s, 0, want[name][0]), want[name][1]) for name, s in spoilt.items()}, dtype)
    p.op.close()
