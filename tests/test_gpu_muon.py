"""Orthogonalised updates (``Muon``) against the same iteration in 64 bits.

Tolerance.  A step's products are off by at most e = 2^-21 + sqrt(K) 2^-24 of the product of their operands' norms (operands of 22 bits, three
of them a step; f32 sums of K terms).  p(s) = a s + b s^3 + c s^5 is odd, so a change of X grows by at most the largest slope of p on [-1.21,
1.21], which is 4.3 (p'(1.21)), a step.  So the result is off by at most sum_k 4.3^(steps - k) e |X_k|, in the Frobenius norm, whose |X_k| the
iteration in 64 bits gives; bf16 results by a half step, 2^-9 of their norm, more."""
import numpy as np
import pytest

import rustingbrain_amd as rb
from rustingbrain_amd import synth
from test_gpu_join import Array

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315


def orthogonalized(u, steps=5):
    """(result, Frobenius bound on the device's error) of one matrix."""
    u = u.astype(np.float64)
    x = u / (np.linalg.norm(u) + 1e-7)
    x = x.T if x.shape[0] > x.shape[1] else x
    e = 2.0 ** -21 + np.sqrt(max(x.shape)) * 2.0 ** -24
    bound = 0.0
    for _ in range(steps):
        bound = 4.3 * (bound + e * np.linalg.norm(x))
        g = x @ x.T
        x = A * x + (B * g + C * g @ g) @ x
    x = x.T if u.shape[0] > u.shape[1] else x
    return x, bound + e * np.linalg.norm(x)


def matrices(count, rows, cols, dtype, seed=0, scale=1e-3):
    rng = np.random.default_rng(rows * 10007 + cols * 13 + count + seed)
    strong = rng.standard_normal((count, rows, 4)) @ rng.standard_normal((count, 4, cols))
    u = (scale * (0.3 * strong + rng.standard_normal((count, rows, cols)))).astype(np.float32)
    return synth.round_bf16(u) if dtype == "bf16" else u


def check(got, u, out_dtype="f32", steps=5):
    for i in range(len(u)):
        want, bound = orthogonalized(u[i], steps)
        if out_dtype == "bf16":
            bound += 2.0 ** -9 * np.linalg.norm(want)
        err = np.linalg.norm(got[i].astype(np.float64) - want)
        assert err <= bound, (i, err, bound, np.linalg.norm(want))


SHAPES = [(1, 1, 1), (2, 1, 7), (3, 5, 1), (2, 31, 33), (3, 32, 32), (2, 33, 64), (4, 64, 31), (2, 65, 130), (3, 130, 66), (5, 96, 224), (2, 227, 341),
          (1, 341, 227), (9, 128, 96), (17, 100, 40), (1, 512, 512), (2, 352, 512), (3, 512, 352), (1, 768, 1408), (1, 1408, 704), (1, 40, 3000),
          (70, 33, 65), (20, 288, 160), (12, 256, 320), (260, 150, 290), (260, 290, 150), (300, 130, 64)]


@pytest.mark.parametrize("count,rows,cols", SHAPES)
def test_orthogonalize(device, count, rows, cols):
    for dtype, out_dtype in (("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")):
        u = matrices(count, rows, cols, dtype)
        m = rb.Muon(device, count, rows, cols)
        src, out = Array(device, u.shape, dtype, u), Array(device, u.shape, out_dtype)
        m.orthogonalize_device(src.ptr, out.ptr, dtype=dtype, out_dtype=out_dtype)
        device.synchronize()
        check(out.get(), u, out_dtype)
        m.close()
        src.free()
        out.free()


def test_the_shapes_reach_every_kernel():
    from rustingbrain_amd import _lib as L
    fn = L.load().rbmoe_internal_muon_tile
    for product in range(3):
        assert {fn(*shape, product) for shape in SHAPES} == {0, 1, 2, 3}, product


def test_singular_values_end_near_one(device):
    u = matrices(2, 200, 300, "f32")
    m = rb.Muon(device, 2, 200, 300)
    a = Array(device, u.shape, "f32", u)
    m.orthogonalize_device(a.ptr, a.ptr)  # in place
    device.synchronize()
    for i in range(2):
        s0 = np.linalg.svd(u[i].astype(np.float64), compute_uv=False)
        s = np.linalg.svd(a.get()[i].astype(np.float64), compute_uv=False)
        assert (s0 / np.linalg.norm(u[i].astype(np.float64))).min() > 0.003
        assert 0.67 <= s.min() and s.max() <= 1.21, (s.min(), s.max())


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 9])
def test_other_numbers_of_steps(device, steps):
    u = matrices(3, 72, 50, "f32")
    m = rb.Muon(device, 3, 72, 50)
    a, o = Array(device, u.shape, "f32", u), Array(device, u.shape, "f32")
    m.orthogonalize_device(a.ptr, o.ptr, steps=steps)
    device.synchronize()
    check(o.get(), u, steps=steps)


def test_sizes_of_numbers(device):
    """Matrices of tiny, huge, zero and spoilt elements in one stack: each by itself."""
    u = matrices(7, 48, 80, "f32", scale=1.0)
    u[0] *= np.float32(1e-30)   # |U| is far below 1e-7: the result is small, not noise
    u[1] *= np.float32(1e18)
    u[2] = 0.0
    u[3, 5, 6] = np.nan
    u[4, 0, 0] = np.inf
    u[5] = 0.0
    u[5, 47, 79] = 2.5          # one element: its own direction
    m = rb.Muon(device, 7, 48, 80)
    a, o = Array(device, u.shape, "f32", u), Array(device, u.shape, "f32")
    m.orthogonalize_device(a.ptr, o.ptr)
    device.synchronize()
    got = o.get()
    for i in (1, 5, 6):
        check(got[i:i + 1], u[i:i + 1])
    assert np.abs(got[0]).max() < 1e-18
    assert (got[2] == 0).all()
    assert np.isnan(got[3]).any() and np.isnan(got[4]).any()
    p = 2.5 / (2.5 + 1e-7)
    for _ in range(5):
        p = A * p + B * p ** 3 + C * p ** 5
    assert abs(got[5, 47, 79] - p) < 1e-5 and (np.delete(got[5].reshape(-1), -1) == 0).all()


def step(w, mo, g, lr, mu, decay, scale, nesterov):
    """One update in 64 bits: (weight, momentum, bound on the weight's Frobenius error beside its rounding)."""
    mo = mu * mo.astype(np.float64) + g
    u = g + mu * mo if nesterov else mo
    o, bound = orthogonalized(u)
    return (1 - lr * decay) * w - lr * scale * o, mo, lr * scale * bound


@pytest.mark.parametrize("count,rows,cols,dtype", [(3, 96, 64, "f32"), (2, 64, 96, "bf16"), (2, 33, 50, "f32"), (1, 130, 70, "bf16"), (4, 352, 512, "f32")])
@pytest.mark.parametrize("nesterov", [True, False])
def test_steps_of_the_optimiser(device, count, rows, cols, dtype, nesterov):
    rng = np.random.default_rng(9)
    lr, mu, decay = 0.02, 0.95, 0.1
    m = rb.Muon(device, count, rows, cols)
    w = rng.standard_normal((count, rows, cols)).astype(np.float32) * np.float32(0.05)
    mo = np.zeros_like(w)
    dw, dm = Array(device, w.shape, "f32", w), Array(device, w.shape, "f32", mo)
    scale = np.sqrt(max(1.0, rows / cols))
    f = np.float32
    for k in range(3):
        g = matrices(count, rows, cols, dtype, seed=k)
        dg = Array(device, g.shape, dtype, g)
        m.step_device(dg.ptr, dm.ptr, dw.ptr, dtype=dtype, lr=lr, momentum=mu, weight_decay=decay, nesterov=nesterov)
        device.synchronize()
        gw, gm = dw.get(), dm.get()
        for i in range(count):
            ww, wm, bound = step(w[i].astype(np.float64), mo[i], g[i].astype(np.float64), float(f(lr)), float(f(mu)), float(f(decay)), scale, nesterov)
            assert np.linalg.norm(gm[i] - wm) <= 2.0 ** -23 * (np.linalg.norm(wm) + np.linalg.norm(mo[i])), k
            # (momentum of the device's own rounding goes into U: 2^-23 of it, a hundredth of the products' part; the decayed weight,
            # its factor and the sum are rounded to 2^-24 each, and the rate to 2^-23)
            assert np.linalg.norm(gw[i] - ww) <= 1.25 * bound + 2.0 ** -22 * np.linalg.norm(ww) + 2.0 ** -22 * lr * scale * np.sqrt(min(rows, cols)) * 1.21, k
        w, mo = gw, gm
        dg.free()


def test_the_same_call_gives_the_same_bits(device):
    u = matrices(6, 150, 90, "f32")
    got = []
    for stack in (u, u):
        m = rb.Muon(device, len(stack), 150, 90)
        a, o = Array(device, stack.shape, "f32", stack), Array(device, stack.shape, "f32")
        m.orthogonalize_device(a.ptr, o.ptr)
        device.synchronize()
        got.append(o.get())
    assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))


def test_refusals(device):
    for count, rows, cols, error in ((0, 4, 4, rb.InvalidConfig), (1, 0, 4, rb.InvalidConfig), (1, 4, -1, rb.InvalidConfig),
                                     (1, 20000, 4, rb.Unsupported), (70000, 4, 4, rb.Unsupported)):
        with pytest.raises(error):
            rb.Muon(device, count, rows, cols)
    m = rb.Muon(device, 1, 8, 8)
    a, b, c = (Array(device, (1, 8, 8), "f32", np.ones((1, 8, 8), np.float32)) for _ in range(3))
    for bad in (dict(steps=0), dict(steps=65), dict(dtype="int8"), dict(out_dtype="int8")):
        with pytest.raises(rb.InvalidConfig):
            m.orthogonalize_device(a.ptr, b.ptr, **bad)
    for i, o in ((0, 1), (1, 0)):
        with pytest.raises(rb.InvalidInput):
            m.orthogonalize_device(i and a.ptr, o and b.ptr)
    with pytest.raises(rb.InvalidInput, match="element"):
        m.orthogonalize_device(a.ptr + 2, b.ptr)
    ok = dict(lr=0.1)
    for bad in (dict(lr=float("nan")), dict(lr=float("inf")), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0),
                dict(weight_decay=float("nan")), dict(update_scale=-1.0), dict(steps=0), dict(dtype="int8")):
        with pytest.raises(rb.InvalidConfig):
            m.step_device(a.ptr, b.ptr, c.ptr, **{**ok, **bad})
    for g, mo, w in ((0, b.ptr, c.ptr), (a.ptr, 0, c.ptr), (a.ptr, b.ptr, 0), (a.ptr, b.ptr, b.ptr), (a.ptr, a.ptr, c.ptr), (a.ptr, b.ptr, a.ptr)):
        with pytest.raises(rb.InvalidInput):
            m.step_device(g, mo, w, **ok)
    device.synchronize()
    assert (a.get() == 1).all() and (b.get() == 1).all() and (c.get() == 1).all()
