"""The operators at the ends of what they accept: offsets beyond 32 bits, more rows than a launch dimension has threads for, the widest rows,
the largest matrices, the most of them."""
import ctypes as C

import numpy as np
import pytest

import rustingbrain_amd as rb
from bench import DeviceBuffer
from rustingbrain_amd import synth
from test_gpu_join import Problem, check_backward, check_forward, stored
from test_gpu_muon import A, B, C as C5, matrices, orthogonalized

pytestmark = pytest.mark.gpu


def bits_of(a, dtype):
    return synth.f32_to_bf16_bits(a) if dtype == "bf16" else np.ascontiguousarray(a, np.float32)


@pytest.mark.parametrize("dtype,gate,rows,cols", [
    ("bf16", "row", (1 << 25) + 5, 64),       # 2^31 elements: a wave a row
    ("bf16", "row", (1 << 20) + 3, 4097),     # 2^32 elements off 16 bytes: a workgroup a row
    ("f32", "row", (1 << 18) + 3, 9001),      # rows read again
    ("f32", "channel", (1 << 20) + 3, 1025),
    ("bf16", "row", (1 << 26) + 5, 8),        # 2^32 threads and more
    ("f32", "row", (1 << 24) + 5, 3)])
def test_the_last_rows_of_a_large_call_are_those_of_a_call_on_them_alone(device, dtype, gate, rows, cols):
    """Every array of both directions, rows of ordinary sizes; the other rows hold whatever the memory holds."""
    tail, es = 9, 2 if dtype == "bf16" else 4
    rng = np.random.default_rng(cols)
    j = rb.ResidualJoin(device, cols, dtype=dtype, gate=gate)
    lib, at, nbytes = device._lib, (rows - tail) * cols * es, tail * cols * es
    big, small, kept = {}, {}, []

    def parameter():
        kept.append(DeviceBuffer(device, cols * 4).upload((1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)))
        return kept[-1].ptr

    try:
        inputs = ["x", "y", "go", "gn"] + (["gate"] if gate == "row" else [])
        outputs = ["out", "normed", "gx", "gy"] + (["gg"] if gate == "row" else [])
        for name in inputs + outputs:
            data = bits_of(stored(rng.standard_normal((tail, cols)), dtype), dtype)
            big[name], small[name] = DeviceBuffer(device, rows * cols * es), DeviceBuffer(device, nbytes).upload(data)
            if name in inputs:
                assert lib.rbmoe_copy_to_device(device.handle, C.c_void_p(big[name].ptr + at), data.ctypes.data_as(C.c_void_p), nbytes) == 0
        post, following = parameter(), parameter()
        channel = parameter() if gate == "channel" else 0
        for n, b in ((tail, small), (rows, big)):
            kw = dict(post_weight_ptr=post, gate_ptr=channel or b["gate"].ptr, next_weight_ptr=following, scale=0.5)
            j.forward_device(n, b["x"].ptr, b["y"].ptr, b["out"].ptr, b["normed"].ptr, **kw)
            j.backward_device(n, b["y"].ptr, b["out"].ptr, b["go"].ptr, b["gn"].ptr, b["gx"].ptr, b["gy"].ptr,
                              grad_gate_ptr=0 if channel else b["gg"].ptr, **kw)
        device.synchronize()
        for name in outputs:
            got, want = (np.empty((tail, cols), np.uint16 if es == 2 else np.uint32) for _ in range(2))
            assert lib.rbmoe_copy_to_host(device.handle, got.ctypes.data_as(C.c_void_p), C.c_void_p(big[name].ptr + at), nbytes) == 0
            small[name].download(want)
            value = synth.bf16_bits_to_f32(want) if es == 2 else want.view(np.float32)
            assert np.isfinite(value).all() and (value != 0).mean() > 0.99, name
            assert np.array_equal(got, want), name
    finally:
        for b in (*big.values(), *small.values(), *kept):
            b.free()
        j.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 70])
def test_the_widest_rows(device, dtype, rows):
    p = Problem(device, rows, 1 << 16, dtype, "channel", padding=rows > 1)
    got = check_forward(p)
    check_backward(p, got.astype(np.float32))
    p.join.close()


def power(v, steps=5):
    for _ in range(steps):
        v = A * v + B * v ** 3 + C5 * v ** 5
    return v


@pytest.mark.parametrize("rows,cols", [(16384, 24), (40, 16384), (16384, 16384)])
def test_the_longest_sides(device, rows, cols):
    """One element a row and column, in a random order: every singular value is an element, and stays alone in its place.  A step on one number
    is off by 2^-21 of it (operands of 22 bits, no sums) and grows what was off by 4.3 at most."""
    n, rng = min(rows, cols), np.random.default_rng(rows + cols)
    r, c = rng.permutation(rows)[:n], rng.permutation(cols)[:n]
    v = (rng.uniform(0.5, 1.5, n) * rng.choice([-1.0, 1.0], n)).astype(np.float32)
    u = np.zeros((rows, cols), np.float32)
    u[r, c] = v
    m = rb.Muon(device, 1, rows, cols)
    a = DeviceBuffer(device, u.nbytes).upload(u)
    m.orthogonalize_device(a.ptr, a.ptr)
    device.synchronize()
    a.download(u)
    x = v.astype(np.float64) / (np.linalg.norm(v.astype(np.float64)) + 1e-7)
    want, bound = power(x), 0.0
    for _ in range(5):
        bound, x = 4.3 * (bound + 2.0 ** -21 * np.abs(x)), power(x, 1)
    assert (np.abs(u[r, c] - want) <= bound + 2.0 ** -21 * np.abs(want)).all()
    u[r, c] = 0.0
    assert not u.any()
    a.free()
    m.close()


def test_the_most_matrices(device):
    count, rows, cols = 65535, 3, 5
    u = matrices(count, rows, cols, "f32")
    m = rb.Muon(device, count, rows, cols)
    a = DeviceBuffer(device, u.nbytes).upload(u)
    m.orthogonalize_device(a.ptr, a.ptr)
    device.synchronize()
    got = a.download(np.empty_like(u))
    for i in (*range(0, count, 97), count - 2, count - 1):
        want, bound = orthogonalized(u[i])
        assert np.linalg.norm(got[i] - want) <= bound, i
    assert np.isfinite(got).all() and (np.abs(got) <= 1.21).all() and (np.abs(got).max(axis=(1, 2)) > 0.1).all()
    a.free()
    m.close()
