"""Rows of infinities, NaN and zeros through a join, backward: each by itself (tolerances: test_gpu_join)."""
import numpy as np
import pytest

from test_gpu_join import Array, Problem, near, stored, unit
from test_gpu_join_range import backward, wanted

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.mark.parametrize("dtype,cols", [("bf16", 768), ("f32", 99), ("bf16", 2047), ("f32", 5000), ("f32", 2), ("bf16", 9000)])
@pytest.mark.parametrize("gate", ["none", "channel", "row"])
@pytest.mark.parametrize("following", [False, True])
def test_without_a_norm_the_gradient_of_y_does_not_depend_on_y(device, dtype, cols, gate, following):
    """grad_y is scale * gate * D: finite, though y is not.  The gate's gradient is y's share and takes what is there."""
    p = Problem(device, 6, cols, dtype, gate, post=False, following=following)
    stream = stored(np.random.default_rng(8).standard_normal((6, cols)), dtype)
    want, size = wanted(p, stream, EPS)
    p.y[1, cols // 2], p.y[2, 0], p.y[3, cols - 1], p.y[4] = np.inf, np.nan, -np.inf, np.nan
    p.d["y"] = Array(device, p.y.shape, dtype, p.y)
    got = backward(p, stream, EPS)
    n = cols / 64 + 40
    for name in ("grad_x", "grad_y"):
        near(got[name], want[name], size[name], n, unit(dtype), name)
    if gate == "row":
        spoilt = ~np.isfinite(p.y)
        assert not np.isfinite(got["grad_gate"][spoilt]).any()
        near(got["grad_gate"][~spoilt], want["grad_gate"][~spoilt], size["grad_gate"][~spoilt], n, unit(dtype), "grad_gate")


@pytest.mark.parametrize("dtype,cols", [("bf16", 768), ("f32", 99), ("bf16", 4096), ("f32", 3), ("bf16", 9000)])
@pytest.mark.parametrize("gate", ["none", "row"])
def test_rows_of_zeros_both_ways(device, dtype, cols, gate):
    """Zero rows of the stream and of the sub-layer: the norms of both are zero, and their gradients 1 / sqrt(eps) times what reaches them."""
    p = Problem(device, 5, cols, dtype, gate)
    p.x[3] = p.y[3] = p.y[1] = 0.0
    p.d["x"], p.d["y"] = Array(device, p.x.shape, dtype, p.x), Array(device, p.y.shape, dtype, p.y)
    out, normed = p.empty(p.x, dtype), p.empty(p.x, dtype)
    p.join.forward_device(5, p.d["x"].ptr, p.d["y"].ptr, out.ptr, normed.ptr, **p.common())
    device.synchronize()
    stream = out.get()
    assert np.array_equal(stream[1], p.x[1]) and (stream[3] == 0).all() and (normed.get()[3] == 0).all()
    assert np.isfinite(stream).all() and np.isfinite(normed.get()).all()
    want, size = wanted(p, stream, EPS)
    got = backward(p, stream, EPS)
    for name in got:
        per_row = want[name].ndim == 2
        near(got[name], want[name], size[name], cols / 64 + 40 + (0 if per_row else 96), unit(dtype if per_row else "f32"), name)
    assert (np.abs(got["grad_y"][3]) > 0).any()


@pytest.mark.parametrize("dtype,cols", [("bf16", 768), ("f32", 99), ("f32", 9000)])
def test_spoilt_rows_behind_a_norm_stay_by_themselves(device, dtype, cols):
    """An infinity or NaN spoils its own row's gradients and the sums over rows, and no other row's."""
    p = Problem(device, 9, cols, dtype, "none")
    stream = stored(np.random.default_rng(8).standard_normal((9, cols)), dtype)
    want, size = wanted(p, stream, EPS)
    p.y[1, 0], p.y[5, cols - 1], stream[7, cols // 2] = np.nan, np.inf, np.nan
    p.d["y"] = Array(device, p.y.shape, dtype, p.y)
    got = backward(p, stream, EPS)
    whole = [0, 2, 3, 4, 6, 8]
    for name in ("grad_x", "grad_y"):
        near(got[name][whole], want[name][whole], size[name][whole], cols / 64 + 40, unit(dtype), name)
    near(got["grad_x"][[1, 5]], want["grad_x"][[1, 5]], size["grad_x"][[1, 5]], cols / 64 + 40, unit(dtype), "grad_x")
    assert np.isnan(got["grad_y"][1]).all() and np.isnan(got["grad_x"][7]).all()
