"""Infinities in the values of a cache come out of ``DecodeAttention`` as the formula has them: one in the result, NaN where two of both signs meet.
(In 8 bits a row with an infinity is NaN whole.)  Tolerances: attention_oracle."""
import numpy as np
import pytest

from test_gpu_kv_cache import Sequences

pytestmark = pytest.mark.gpu
INF = np.inf


@pytest.mark.parametrize("dtype,longest", [("bf16", 300), ("f32", 300), ("bf16", 3000), ("f32", 3000)])
def test_infinite_values_in_a_cache(device, dtype, longest):
    s = Sequences(device, [300, 40, 7], (8, 2, 64), 16, dtype, dtype)
    place = lambda i, at: int(s.tables[i, at // 16]) * 16 + at % 16  # noqa: E731
    k, v = (s.c.kept[j].copy() for j in range(2))
    clean = s.run(longest=longest)
    v[place(0, 33), 1, 5], v[place(0, 299), 1, 6], v[place(1, 39), 0, 63], v[place(2, 0), 0, 0], v[place(2, 6), 0, 0] = INF, -INF, -INF, INF, -INF
    kept = s.c.kept.copy()
    s.c.write(k, v, np.arange(len(v)))
    got = s.run(longest=longest)
    for i, heads, col, value in ((0, slice(4, 8), 5, INF), (0, slice(4, 8), 6, -INF), (1, slice(0, 4), 63, -INF)):
        assert (got[i, heads, col] == value).all(), (i, col, got[i, heads, col])
        got[i, heads, col] = clean[i, heads, col]
    assert np.isnan(got[2, :4, 0]).all()
    got[2, :4, 0] = clean[2, :4, 0]
    s.c.kept = kept
    s.check(got)
    s.op.close()
    s.c.op.close()
