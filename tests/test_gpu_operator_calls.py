"""The operators around the layer called the ways a program calls them: captured and replayed, on a stream of the caller's own, together
in one step, over arrays whose offsets pass 32 bits, and with the device handle given up first."""
import ctypes as C

import numpy as np
import pytest

import rustingbrain_amd as rb
from bench import DeviceBuffer
from test_gpu_graph import Capture, hip  # noqa: F401  (a fixture)
from test_gpu_join import Array
from test_gpu_muon import matrices

pytestmark = pytest.mark.gpu


class Step:
    """Join forward and backward and two updates that take its parameters' neighbours: a linear sub-layer's weight stack."""

    def __init__(self, device, rows=300, cols=256, seed=1):
        rng = np.random.default_rng(seed)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        A = lambda a, t="bf16": Array(device, a.shape, t, a)  # noqa: E731
        self.rows, self.device = rows, device
        self.x, self.y, self.go, self.gn = (A(f(rows, cols)) for _ in range(4))
        self.post, self.gate, self.next = (A(1 + 0.1 * f(cols), "f32") for _ in range(3))
        self.out, self.normed, self.gx, self.gy = (Array(device, (rows, cols), "bf16") for _ in range(4))
        self.gp, self.gg, self.gnx = (A(np.zeros(cols, np.float32), "f32") for _ in range(3))
        self.join = rb.ResidualJoin(device, cols, dtype="bf16", gate="channel")
        self.muon = rb.Muon(device, 3, 96, 160)
        self.grad, self.momentum, self.weight = (A(f(3, 96, 160) * 1e-2, "f32") for _ in range(3))
        self.tall = rb.Muon(device, 2, 130, 50)
        self.u, self.o = A(matrices(2, 130, 50, "bf16")), Array(device, (2, 130, 50), "bf16")

    def run(self):
        kw = dict(post_weight_ptr=self.post.ptr, gate_ptr=self.gate.ptr, next_weight_ptr=self.next.ptr, scale=0.5)
        self.join.forward_device(self.rows, self.x.ptr, self.y.ptr, self.out.ptr, self.normed.ptr, **kw)
        self.join.backward_device(self.rows, self.y.ptr, self.out.ptr, self.go.ptr, self.gn.ptr, self.gx.ptr, self.gy.ptr,
                                  grad_post_ptr=self.gp.ptr, grad_gate_ptr=self.gg.ptr, grad_next_ptr=self.gnx.ptr, accumulate=True, **kw)
        self.muon.step_device(self.grad.ptr, self.momentum.ptr, self.weight.ptr, lr=0.02, weight_decay=0.1)
        self.tall.orthogonalize_device(self.u.ptr, self.o.ptr, dtype="bf16", out_dtype="bf16")

    def results(self):
        self.device.synchronize()
        return [a.get() for a in (self.out, self.normed, self.gx, self.gy, self.gp, self.gg, self.gnx, self.momentum, self.weight, self.o)]


def same(a, b):
    return all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(a, b))


def test_a_captured_step_replays_like_the_eager_one(device, hip):  # noqa: F811
    eager, captured = Step(device), Step(device)
    cap = Capture(hip, device, captured.run)
    for _ in range(4):
        device.set_stream(None)
        eager.run()
        want = eager.results()
        cap.replay()
        assert same(captured.results(), want)
    cap.close()


def test_on_a_stream_of_the_callers_own(device, hip):  # noqa: F811
    a, b = Step(device), Step(device)
    a.run()
    want = a.results()
    stream = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    try:
        device.set_stream(stream.value)
        b.run()
        got = b.results()  # (waits for the stream that the calls were given)
    finally:
        device.set_stream(None)
        hip.hipStreamDestroy(stream)
    assert same(got, want)


def last_rows_are_those_of_a_call_on_them_alone(device, rows, cols):
    tail = 9
    j = rb.ResidualJoin(device, cols, dtype="bf16")
    rng = np.random.default_rng(0)
    bits = lambda: (rng.integers(0, 1 << 15, (tail, cols)) % 0x3f80 + 0x3f00).astype(np.uint16)  # noqa: E731
    big, small = [], []
    at = (rows - tail) * cols * 2
    lib = device._lib
    try:
        for i in range(4):
            big.append(DeviceBuffer(device, rows * cols * 2))
            small.append(DeviceBuffer(device, tail * cols * 2))
            data = bits()
            small[-1].upload(data)
            assert lib.rbmoe_copy_to_device(device.handle, C.c_void_p(big[-1].ptr + at), data.ctypes.data_as(C.c_void_p), data.nbytes) == 0
        w = DeviceBuffer(device, cols * 4).upload(np.linspace(0.5, 1.5, cols).astype(np.float32))
        for n, b in ((rows, big), (tail, small)):
            j.forward_device(n, b[0].ptr, b[1].ptr, b[2].ptr, b[3].ptr, post_weight_ptr=w.ptr, next_weight_ptr=w.ptr)
            j.backward_device(n, b[1].ptr, b[2].ptr, b[3].ptr, 0, b[0].ptr, b[3].ptr, post_weight_ptr=w.ptr)
        device.synchronize()
        for i in range(4):
            got, want = np.empty((tail, cols), np.uint16), np.empty((tail, cols), np.uint16)
            assert lib.rbmoe_copy_to_host(device.handle, got.ctypes.data_as(C.c_void_p), C.c_void_p(big[i].ptr + at), got.nbytes) == 0
            small[i].download(want)
            assert np.array_equal(got, want), i
    finally:
        for b in big + small:
            b.free()


def test_offsets_beyond_32_bits(device):
    """Rows of 4.3 GB each way."""
    last_rows_are_those_of_a_call_on_them_alone(device, (1 << 25) + 5, 64)


@pytest.mark.parametrize("rows,cols", [((1 << 26) + 5, 8), ((1 << 24) + 5, 3)])
def test_more_rows_than_a_dimension_of_a_launch_has_threads_for(device, rows, cols):
    """A row takes a wave, or where it is shorter than 16 bytes a workgroup."""
    last_rows_are_those_of_a_call_on_them_alone(device, rows, cols)


def test_an_operator_outlives_its_device_handle():
    dev = rb.Device.open(0)
    j, m = rb.ResidualJoin(dev, 64), rb.Muon(dev, 1, 8, 8)
    dev.close()
    j.close()
    m.close()
