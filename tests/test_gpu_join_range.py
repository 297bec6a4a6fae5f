"""The backward pass of a join over rows far from one in size, and rows of zeros, against the formulas in 64 bits (tolerances: test_gpu_join)."""
import numpy as np
import pytest

import join_oracle as jo
from test_gpu_join import Array, Problem, near, ptr, stored, unit

pytestmark = pytest.mark.gpu


def backward(p, stream, eps):
    """The device's gradients of a problem whose `out` is `stream`, by name."""
    names = [("grad_x", p.x, p.dtype), ("grad_y", p.x, p.dtype), ("grad_post", p.post, "f32"),
             ("grad_gate", p.gate, "f32" if p.gate_mode == "channel" else p.dtype), ("grad_next", p.next, "f32")]
    arrays = {name: p.empty(like, t) for name, like, t in names if like is not None}
    p.join.backward_device(p.rows, p.d["y"].ptr, Array(p.dev, stream.shape, p.dtype, stream).ptr if p.next is not None else 0, p.d["go"].ptr,
                           ptr(p.d["gn"]), arrays["grad_x"].ptr, arrays["grad_y"].ptr,
                           **{name + "_ptr": ptr(arrays.get(name)) for name in ("grad_post", "grad_gate", "grad_next")},
                           **{**p.common(), "eps": eps})
    p.dev.synchronize()
    return {name: a.get().astype(np.float64) for name, a in arrays.items()}


def wanted(p, stream, eps):
    wide = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    return jo.backward(wide(p.y), wide(stream), p.live, wide(p.post), wide(p.gate), p.scale, wide(p.next), eps, wide(p.go), wide(p.gn),
                       p.gate_mode == "channel")


def scaled(p, rows_by):
    """The problem with rows of y of these sizes, and rows for `out` of the same."""
    rng = np.random.default_rng(8)
    p.y, out = (stored(rng.standard_normal(p.y.shape) * rows_by[:, None], p.dtype) for _ in range(2))
    p.d["y"] = Array(p.dev, p.y.shape, p.dtype, p.y)
    return out


@pytest.mark.parametrize("dtype,cols", [("f32", 96), ("bf16", 768), ("f32", 1365), ("bf16", 4096), ("f32", 3), ("f32", 9000), ("bf16", 9001)])
@pytest.mark.parametrize("gate", ["channel", "row"])
@pytest.mark.parametrize("eps,sizes", [(1e-6, [1.0, 1e4, 1e9, 1e12, 1e13, 1e14, 1e15, 1e16, 0.0, 1e-8]),
                                       # (a norm of rows alone: nothing beside the squares, which f32 holds down to rows of 1e-18)
                                       (0.0, [1.0, 1e-6, 1e-10, 1e-13, 1e-14, 1e-16, 1e10, 1e16]),
                                       # an eps whose inverse root's cube passes f32's range, and rows of zeros
                                       (1e-30, [1.0, 0.0, 1e-14, 1e-16, 1e16])])
def test_rows_of_every_size(device, dtype, cols, gate, eps, sizes):
    """A gradient is what a row's projection leaves of it times its inverse RMS, whatever the RMS is."""
    p = Problem(device, len(sizes), cols, dtype, gate)
    stream = scaled(p, np.array(sizes, np.float64))
    got = backward(p, stream, eps)
    want, size = wanted(p, stream, float(np.float32(eps)))
    n = p.cols / 64 + 40
    for name in got:
        assert np.isfinite(want[name]).all(), name
        per_row = want[name].ndim == 2
        near(got[name], want[name], size[name], n + (0 if per_row else p.rows / 256 + 96),
             unit(p.dtype if per_row else "f32"), name)
