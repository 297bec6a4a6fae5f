"""How exact orthogonalised updates are: of matrices of every size of numbers, beside the same iteration in f32.

Tolerance.  The device's products round their operands to 22 bits, two fewer than f32 has, and add up in f32: so the result may be four times
as far from the iteration in 64 bits as the one in f32 (numpy) is on the same input, in the Frobenius norm.  A matrix of a few elements may be
exact by chance in f32, so 2^-18 of the result's norm is let pass anyway: five steps magnify a relative error by 4.3^5 / 3.4^5 = 3.1 at
most while they grow a singular value and each adds roundings of a few 2^-23.  Operands of 16 bits (two bf16 numbers) end two to fourteen times
above this on the matrices below, of 11 bits two hundred times."""
import numpy as np
import pytest

import rustingbrain_amd as rb
from test_gpu_join import Array
from test_gpu_muon import A, B, C, matrices, orthogonalized

pytestmark = pytest.mark.gpu


def in_f32(u, steps):
    f = np.float32
    x = (u / f(np.linalg.norm(u.astype(np.float64)) + 1e-7)).astype(f)
    x = np.ascontiguousarray(x.T) if x.shape[0] > x.shape[1] else x
    for _ in range(steps):
        g = x @ x.T
        x = f(A) * x + (f(B) * g + f(C) * (g @ g)) @ x
    return x.T if u.shape[0] > u.shape[1] else x


def as_exact_as_f32(got, u, steps=5):
    for i in range(len(u)):
        want, _ = orthogonalized(u[i], steps)
        err, f32 = (np.linalg.norm(v.astype(np.float64) - want) for v in (got[i], in_f32(u[i], steps)))
        assert err <= max(4 * f32, 2.0 ** -18 * np.linalg.norm(want)), (i, err, f32, np.linalg.norm(want))


@pytest.mark.parametrize("steps", [1, 5, 8])
@pytest.mark.parametrize("count,rows,cols", [(9, 48, 80), (9, 130, 70), (18, 256, 160), (99, 160, 224), (260, 150, 290)])
def test_sizes_of_numbers(device, count, rows, cols, steps):
    """A matrix far below the 1e-7 of the divisor comes out small, and as exact as any: its error is held to a share of its own norm."""
    u = matrices(count, rows, cols, "f32", scale=1.0)
    for i, s in enumerate((1e-36, 1e-30, 1e-20, 1e-14, 1e-12, 1e-10, 1e-9, 1e-8, 1e-7)):
        u[i] *= np.float32(s)
    m = rb.Muon(device, count, rows, cols)
    a, o = Array(device, u.shape, "f32", u), Array(device, u.shape, "f32")
    m.orthogonalize_device(a.ptr, o.ptr, steps=steps)
    device.synchronize()
    as_exact_as_f32(o.get(), u, steps)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("count,rows,cols", [(1, 1, 1), (3, 5, 1), (2, 31, 33), (2, 227, 341), (9, 128, 96), (1, 512, 512), (2, 352, 512), (1, 768, 1408),
                                             (1, 1408, 704), (1, 40, 3000), (1, 16000, 17), (70, 33, 65), (40, 288, 160), (260, 150, 290)])
def test_ordinary_matrices(device, count, rows, cols, dtype):
    u = matrices(count, rows, cols, dtype)
    m = rb.Muon(device, count, rows, cols)
    a, o = Array(device, u.shape, dtype, u), Array(device, u.shape, "f32")
    m.orthogonalize_device(a.ptr, o.ptr, dtype=dtype)
    device.synchronize()
    as_exact_as_f32(o.get(), u)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_steps_on_momentum_that_has_decayed(device, dtype):
    """What is left of the momentum of an expert that gets no tokens: gradients of zero."""
    count, rows, cols = 4, 96, 160
    lr, mu = 0.5, 0.9
    m = rb.Muon(device, count, rows, cols)
    w = np.zeros((count, rows, cols), np.float32)  # (so that the weight is the update alone)
    mo = matrices(count, rows, cols, "f32", scale=1.0) * np.array([1e-3, 1e-9, 1e-12, 1e-20], np.float32)[:, None, None]
    g = np.zeros_like(w)
    dw, dm, dg = Array(device, w.shape, "f32", w), Array(device, w.shape, "f32", mo), Array(device, g.shape, dtype, g)
    m.step_device(dg.ptr, dm.ptr, dw.ptr, dtype=dtype, lr=lr, momentum=mu)
    device.synchronize()
    u = dm.get() * np.float32(mu)  # (the device's momentum: G = 0 leaves mu M of the direction)
    as_exact_as_f32(dw.get() / np.float32(-lr), u)
