"""A sub-layer joined to the residual stream (``ResidualJoin``) against the same formulas in 64 bits.

Tolerances.  An output is rounded once: at most u |value|, u = 2^-24 (f32) or 2^-8 (bf16, taken as a whole step).  In front of that
rounding stand f32 operations.  A row's sum of d squares or products is taken by lanes that add up to ceil(d / 64) terms and six to eight
more between them; a workgroup's sum over rows adds at most ceil(rows / (parts * rows a turn)) + 3 + parts / 8 + 8 terms.  Each addition
and each of the dozen operations beside it is off by 2^-24 of the magnitudes it adds, so the bound is
N * 2^-24 * (sum of the magnitudes), with N the number of operations in a row."""
import ctypes as C

import numpy as np
import pytest

import join_oracle as jo
import rustingbrain_amd as rb
from bench import DeviceBuffer
from rustingbrain_amd import _lib as L
from rustingbrain_amd import synth

pytestmark = pytest.mark.gpu
EPS = 1e-6
PAD = 256  # bytes in front of and behind every array, which no call may change


class Array:
    """A device array between two guards, from any element on."""

    def __init__(self, dev, shape, dtype, data=None, shift=0):
        self.shape, self.dtype = shape, dtype
        self.es = 2 if dtype == "bf16" else (1 if dtype == "u8" else 4)
        self.n = int(np.prod(shape))
        self.buf = DeviceBuffer(dev, self.n * self.es + 2 * PAD + 64)
        self.at = PAD + shift * self.es
        raw = np.full(self.buf.nbytes, 0xA5, np.uint8)
        if data is not None:
            bits = synth.f32_to_bf16_bits(np.asarray(data, np.float32)) if dtype == "bf16" else np.asarray(data)
            raw[self.at:self.at + self.n * self.es] = np.ascontiguousarray(bits).reshape(-1).view(np.uint8)
        self.buf.upload(raw)

    @property
    def ptr(self):
        return self.buf.ptr + self.at

    def get(self):
        raw = self.buf.download(np.empty(self.buf.nbytes, np.uint8))
        assert (raw[:self.at] == 0xA5).all() and (raw[self.at + self.n * self.es:] == 0xA5).all(), "bytes beside the array changed"
        body = raw[self.at:self.at + self.n * self.es].copy()
        if self.dtype == "bf16":
            return synth.bf16_bits_to_f32(body.view(np.uint16)).reshape(self.shape)
        return body.view(np.float32).reshape(self.shape)

    def free(self):
        self.buf.free()


def stored(a, dtype):
    a = np.asarray(a, np.float32)
    return synth.round_bf16(a) if dtype == "bf16" else a


def ptr(a):
    return 0 if a is None else a.ptr


class Problem:
    def __init__(self, dev, rows, cols, dtype, gate, post=True, following=True, padding=False, shift=0, seed=0, scale=0.3):
        rng = np.random.default_rng(1000 * rows + cols + seed)
        self.rows, self.cols, self.dtype, self.gate_mode, self.scale = rows, cols, dtype, gate, scale
        row = lambda std: stored(std * rng.standard_normal((rows, cols)), dtype)  # noqa: E731
        self.x, self.y = row(2.0), stored(rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, 1))), dtype)
        self.live = np.ones(rows, bool)
        if padding:
            self.live[rng.permutation(rows)[:max(1, rows // 4)]] = False
            self.y[~self.live] = np.nan
        f32 = lambda c, s: (c + s * rng.standard_normal(cols)).astype(np.float32)  # noqa: E731
        self.post = f32(1.0, 0.1) if post else None
        self.next = f32(1.0, 0.1) if following else None
        self.gate = None if gate == "none" else f32(0.5, 0.2) if gate == "channel" else row(1.0)
        if gate == "row" and padding:
            self.gate[~self.live] = np.inf
        self.go, self.gn = row(0.1), row(0.1) if following else None
        self.dev = dev
        a = lambda v, t=dtype: None if v is None else Array(dev, v.shape, t, v, shift)  # noqa: E731
        self.d = dict(x=a(self.x), y=a(self.y), go=a(self.go), gn=a(self.gn), post=a(self.post, "f32"), next=a(self.next, "f32"),
                      gate=a(self.gate, "f32" if gate == "channel" else dtype),
                      valid=a(self.live.astype(np.uint8), "u8") if padding else None)
        self.empty = lambda like, t: None if like is None else Array(dev, like.shape, t, None, shift)
        self.join = rb.ResidualJoin(dev, cols, dtype=dtype, gate=gate)

    def common(self):
        d = self.d
        return dict(valid_ptr=ptr(d["valid"]), post_weight_ptr=ptr(d["post"]), gate_ptr=ptr(d["gate"]),
                    next_weight_ptr=ptr(d["next"]), scale=self.scale, eps=EPS)

    def wide(self):
        w = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
        return w(self.post), w(self.gate), w(self.next)


def unit(dtype):
    return 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24


def near(got, want, magnitude, operations, u, what):
    bound = u * np.abs(want) + operations * 2.0 ** -24 * magnitude + 1e-37
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4], bound[bad][:4])


def check_forward(p, in_place=False):
    out = p.d["x"] if in_place else p.empty(p.x, p.dtype)
    normed = (p.d["y"] if in_place else p.empty(p.x, p.dtype)) if p.next is not None else None
    p.join.forward_device(p.rows, p.d["x"].ptr, p.d["y"].ptr, out.ptr, ptr(normed), **p.common())
    p.dev.synchronize()
    post, gate, following = p.wide()
    x = p.x.astype(np.float64)
    b = jo.branch(p.y.astype(np.float64), p.live, post, gate, p.scale, EPS)
    got = out.get().astype(np.float64)
    n = p.cols / 64 + 24
    near(got, x + b, np.abs(x) + np.abs(b), n, unit(p.dtype), "out")
    if normed is not None:
        want = jo.rms_norm(got, EPS) * following  # of the rows as stored
        near(normed.get().astype(np.float64), want, np.abs(want), n, unit(p.dtype), "normed")
    return got


def check_backward(p, stream, accumulate=False):
    names = [("grad_x", p.x, p.dtype), ("grad_y", p.x, p.dtype), ("grad_post", p.post, "f32"),
             ("grad_gate", p.gate, "f32" if p.gate_mode == "channel" else p.dtype), ("grad_next", p.next, "f32")]
    before = {}
    arrays = {}
    for name, like, t in names:
        if like is None:
            arrays[name] = None
            continue
        before[name] = np.random.default_rng(5).standard_normal(like.shape).astype(np.float32) if like.ndim == 1 and accumulate else None
        arrays[name] = Array(p.dev, like.shape, t, before[name], 0) if before[name] is not None else p.empty(like, t)
    out = Array(p.dev, p.x.shape, p.dtype, stream)
    p.join.backward_device(p.rows, p.d["y"].ptr, out.ptr if p.next is not None else 0, p.d["go"].ptr, ptr(p.d["gn"]),
                           arrays["grad_x"].ptr, arrays["grad_y"].ptr, grad_post_ptr=ptr(arrays["grad_post"]),
                           grad_gate_ptr=ptr(arrays["grad_gate"]), grad_next_ptr=ptr(arrays["grad_next"]), accumulate=accumulate,
                           **p.common())
    p.dev.synchronize()
    post, gate, following = p.wide()
    gn = None if p.gn is None else p.gn.astype(np.float64)
    want, size = jo.backward(p.y.astype(np.float64), stream.astype(np.float64), p.live, post, gate, p.scale, following, EPS,
                             p.go.astype(np.float64), gn, p.gate_mode == "channel")
    n = p.cols / 64 + 40
    got = {}
    for name, like, t in names:
        if like is None:
            continue
        got[name] = arrays[name].get()
        per_row = like.ndim == 2
        w, m = want[name], size[name]
        if before[name] is not None:
            w, m = w + before[name], m + np.abs(before[name])
        near(got[name].astype(np.float64), w, m, n + (0 if per_row else p.rows / 256 + 96), unit(t), name)
    return got


SHAPES = [(1, 512), (1, 1), (2, 3), (5, 64), (3, 65), (7, 130), (33, 227), (9, 514), (66, 512), (130, 760), (17, 1024), (5, 1365), (6, 1366),
          (4, 2048), (3, 2050), (5, 4096), (2, 5001), (3, 8192), (2, 8200), (2, 20000)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype,gate", [("f32", "none"), ("f32", "row"), ("bf16", "channel"), ("bf16", "row")])
def test_both_ways(device, rows, cols, dtype, gate):
    p = Problem(device, rows, cols, dtype, gate, padding=rows > 2)
    got = check_forward(p)
    check_backward(p, got.astype(np.float32))


@pytest.mark.parametrize("gate", ["none", "channel", "row"])
@pytest.mark.parametrize("post,following", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype,cols", [("bf16", 768), ("f32", 99), ("bf16", 9000)])
def test_norms_left_out(device, dtype, cols, post, following, gate):
    p = Problem(device, 21, cols, dtype, gate, post=post, following=following, padding=True)
    got = check_forward(p)
    check_backward(p, got.astype(np.float32))


@pytest.mark.parametrize("dtype,cols,shift", [("bf16", 512, 1), ("bf16", 512, 2), ("bf16", 512, 4), ("f32", 256, 1), ("f32", 256, 2),
                                              ("bf16", 4096, 3)])
def test_rows_from_any_element_on(device, dtype, cols, shift):
    p = Problem(device, 11, cols, dtype, "row", shift=shift)
    got = check_forward(p)
    check_backward(p, got.astype(np.float32))


# (rows end 1 to 7 elements into their last 16 bytes, whatever they start on)
@pytest.mark.parametrize("dtype,cols", [("bf16", c) for c in [*range(7, 17), *range(1017, 1032), 2049, 2055]] +
                                       [("f32", c) for c in [*range(3, 9), *range(1021, 1029), 2050]])
def test_rows_that_end_inside_a_vector(device, dtype, cols):
    p = Problem(device, 9, cols, dtype, "row", padding=True, shift=cols % 3)
    got = check_forward(p)
    check_backward(p, got.astype(np.float32))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype,cols", [("bf16", 515), ("bf16", 1029), ("bf16", 4095), ("f32", 1023), ("f32", 2050), ("f32", 4093),
                                        ("bf16", 6000), ("bf16", 8191), ("f32", 5000), ("f32", 8189)])
def test_in_place_and_accumulated_at_odd_widths(device, dtype, cols, rows):
    p = Problem(device, rows, cols, dtype, "channel", padding=rows > 1, shift=1)
    stream = stored(np.random.default_rng(8).standard_normal((rows, cols)), dtype)
    check_backward(p, stream, accumulate=True)
    check_forward(p, in_place=True)


@pytest.mark.parametrize("dtype,cols", [("bf16", 1024), ("f32", 300), ("f32", 9001)])
def test_in_place_and_accumulated(device, dtype, cols):
    p = Problem(device, 40, cols, dtype, "channel", padding=True)
    stream = stored(np.random.default_rng(8).standard_normal((40, cols)), dtype)
    check_backward(p, stream, accumulate=True)
    check_forward(p, in_place=True)


@pytest.mark.parametrize("dtype,cols", [("bf16", 1024), ("f32", 300), ("f32", 9001)])
def test_input_gradients_may_take_the_place_of_what_they_are_made_from(device, dtype, cols):
    p = Problem(device, 21, cols, dtype, "row", padding=True)
    stream = stored(np.random.default_rng(8).standard_normal((21, cols)), dtype)
    apart = check_backward(p, stream)
    out, gate = Array(device, stream.shape, dtype, stream), p.empty(p.x, dtype)
    p.join.backward_device(21, p.d["y"].ptr, out.ptr, p.d["go"].ptr, p.d["gn"].ptr, p.d["go"].ptr, p.d["gn"].ptr, grad_gate_ptr=gate.ptr,
                           **p.common())
    device.synchronize()
    assert np.array_equal(p.d["go"].get(), apart["grad_x"]) and np.array_equal(p.d["gn"].get(), apart["grad_y"])
    assert np.array_equal(gate.get(), apart["grad_gate"])


def test_parts_of_the_backward_pass_left_out(device):
    """No gradient of a parameter wanted, and none behind the add: the others are what they are with them."""
    p = Problem(device, 33, 512, "bf16", "channel")
    stream = stored(np.random.default_rng(8).standard_normal((33, 512)), "bf16")
    whole = check_backward(p, stream)
    out = Array(device, stream.shape, "bf16", stream)
    gx, gy, zeros = p.empty(p.x, "bf16"), p.empty(p.x, "bf16"), Array(device, p.x.shape, "bf16", np.zeros_like(p.x))
    p.join.backward_device(33, p.d["y"].ptr, out.ptr, p.d["go"].ptr, p.d["gn"].ptr, gx.ptr, gy.ptr, **p.common())
    device.synchronize()
    assert np.array_equal(gx.get(), whole["grad_x"]) and np.array_equal(gy.get(), whole["grad_y"])
    got = []
    for go in (0, zeros.ptr):
        p.join.backward_device(33, p.d["y"].ptr, out.ptr, go, p.d["gn"].ptr, gx.ptr, gy.ptr, **p.common())
        device.synchronize()
        got.append((gx.get(), gy.get()))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])


def test_more_rows_than_one_round_of_workgroups(device):
    for dtype, rows, cols in (("bf16", 5003, 512), ("f32", 2500, 96), ("bf16", 700, 3000)):
        p = Problem(device, rows, cols, dtype, "channel", padding=True)
        got = check_forward(p)
        first = check_backward(p, got.astype(np.float32))
        again = check_backward(p, got.astype(np.float32))
        for name in first:
            assert np.array_equal(first[name].view(np.uint32), again[name].view(np.uint32)), name


def test_rows_of_zeros_infinities_and_nan_stay_by_themselves(device):
    p = Problem(device, 6, 512, "f32", "none")
    p.y[0] = 0.0
    p.y[1, 5] = np.inf
    p.y[2, 7] = np.nan
    p.x[3] = -p.scale * 0.0
    q = Array(device, p.y.shape, "f32", p.y)
    out, normed = p.empty(p.x, "f32"), p.empty(p.x, "f32")
    p.join.forward_device(6, p.d["x"].ptr, q.ptr, out.ptr, normed.ptr, **p.common())
    device.synchronize()
    got, n = out.get(), normed.get()
    assert np.array_equal(got[0], p.x[0])            # the norm of a row of zeros is zero, not NaN
    assert np.isnan(got[1, 5]) and np.isnan(got[2]).all()
    assert np.isfinite(got[[0, 3, 4, 5]]).all() and np.isfinite(n[[0, 3, 4, 5]]).all()


def test_no_rows(device):
    j = rb.ResidualJoin(device, 64, dtype="f32", gate="channel")
    j.forward_device(0, 0, 0, 0)
    g = [Array(device, (64,), "f32", np.full(64, 3.0, np.float32)) for _ in range(3)]
    kw = dict(grad_post_ptr=g[0].ptr, grad_gate_ptr=g[1].ptr, grad_next_ptr=g[2].ptr)
    j.backward_device(0, 0, 0, 0, 0, 0, 0, accumulate=True, **kw)
    device.synchronize()
    assert all((a.get() == 3.0).all() for a in g)
    j.backward_device(0, 0, 0, 0, 0, 0, 0, **kw)
    device.synchronize()
    assert all((a.get() == 0.0).all() for a in g)


def test_refusals(device):
    p = Problem(device, 4, 64, "bf16", "channel")
    d, out = p.d, p.empty(p.x, "bf16")
    ok = dict(p.common())
    fwd = lambda **kw: p.join.forward_device(4, d["x"].ptr, d["y"].ptr, out.ptr, kw.pop("normed", 0), **{**ok, "next_weight_ptr": 0, **kw})  # noqa: E731
    fwd()
    for bad in (dict(gate_ptr=0), dict(normed=d["go"].ptr), dict(next_weight_ptr=d["next"].ptr), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(eps=-1.0), dict(eps=float("nan")), dict(post_weight_ptr=d["post"].ptr + 2),
                dict(normed=out.ptr, next_weight_ptr=d["next"].ptr)):
        with pytest.raises(rb.InvalidInput):
            fwd(**bad)
    with pytest.raises(rb.Unsupported):
        p.join.forward_device((1 << 30) + 1, d["x"].ptr, d["y"].ptr, out.ptr, **{**ok, "next_weight_ptr": 0})
    for rows, x, y, o in ((-1, 1, 1, 1), (4, 0, 1, 1), (4, 1, 0, 1), (4, 1, 1, 0)):
        with pytest.raises(rb.InvalidInput):
            p.join.forward_device(rows, x and d["x"].ptr, y and d["y"].ptr, o and out.ptr, **{**ok, "next_weight_ptr": 0})
    with pytest.raises(rb.InvalidInput, match="element"):
        p.join.forward_device(4, d["x"].ptr + 1, d["y"].ptr, out.ptr, **{**ok, "next_weight_ptr": 0})
    g = [p.empty(p.x, "bf16") for _ in range(2)]
    back = lambda **kw: p.join.backward_device(  # noqa: E731
        4, kw.pop("y", d["y"].ptr), kw.pop("out", out.ptr), kw.pop("go", d["go"].ptr), kw.pop("gn", d["gn"].ptr),
        kw.pop("gx", g[0].ptr), kw.pop("gy", g[1].ptr), **{**ok, **kw})
    back()
    for bad in (dict(y=0), dict(out=0), dict(gn=0), dict(gx=0), dict(gy=0), dict(gy=g[0].ptr), dict(go=0, gn=0, next_weight_ptr=0),
                dict(post_weight_ptr=0, grad_post_ptr=g[0].ptr), dict(next_weight_ptr=0, gn=0, grad_next_ptr=g[0].ptr)):
        with pytest.raises(rb.InvalidInput):
            back(**bad)
    plain = rb.ResidualJoin(device, 64, dtype="bf16")
    with pytest.raises(rb.InvalidInput, match="without a gate"):
        plain.forward_device(4, d["x"].ptr, d["y"].ptr, out.ptr, gate_ptr=d["gate"].ptr)
    device.synchronize()
    for cols, dtype, gate, error in ((0, "f32", "none", rb.InvalidConfig), (70000, "f32", "none", rb.Unsupported),
                                     (8, "int8", "none", rb.InvalidConfig)):
        with pytest.raises(error):
            rb.ResidualJoin(device, cols, dtype=dtype, gate=gate)
    lib = L.load()
    h = C.c_void_p()
    assert lib.rbmoe_join_create(device.handle, 8, 2, 0, C.byref(h)) == L.INVALID_CONFIG
    assert lib.rbmoe_join_create(device.handle, 8, 0, 3, C.byref(h)) == L.INVALID_CONFIG


def test_the_budget_counts_the_workspace():
    small = rb.Device.open(0, 1)
    try:
        with pytest.raises(rb.MemoryBudget):
            rb.ResidualJoin(small, 1024)
        with pytest.raises(rb.MemoryBudget):
            rb.Muon(small, 4, 512, 512)
        j = rb.ResidualJoin(small, 16)
        j.close()
    finally:
        small.close()
