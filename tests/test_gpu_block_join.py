"""The block step with a norm behind the layer, a gate and a residual scale (``MoeLayer.set_block_join``), against the oracle's layer and
the join's formulas in 64 bits.  Tolerances: the layer's own bars (rel-L2 1e-5 all-f32, 2e-2 bf16) for the output; gradients pass three
stages that are within that bar each (join, layer, norm), so three times it in f32."""
import ctypes as C

import numpy as np
import pytest

import join_oracle as jo
import rustingbrain_amd as rb
from bench import DeviceBuffer
from conftest import rel_l2
from helpers import gpu_layer, oracle_layer, small_workload, tolerance
from oracle import rb_oracle as orc
from rustingbrain_amd import _lib as L
from rustingbrain_amd import synth
from test_gpu_graph import Capture, hip  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
EPS = 1e-6


class Block:
    def __init__(self, device, shape, act, wt, post=True, gate=True, scale=0.4, training=False, padding=False, seed=71):
        self.t = synth.make(small_workload(seed=seed, act=act, wt=wt, **shape))
        rng = np.random.default_rng(seed)
        d, T = shape["d"], shape["T"]
        self.bf16 = act == "bf16"
        self.stored = synth.round_bf16 if self.bf16 else (lambda a: np.asarray(a, np.float32))
        self.norm = rng.uniform(0.5, 1.5, d).astype(np.float32)
        self.post = rng.uniform(0.5, 1.5, d).astype(np.float32) if post else None
        self.gate = rng.uniform(-1.0, 1.0, d).astype(np.float32) if gate else None
        self.scale = scale
        self.live = np.ones(T, bool)
        if padding:
            self.live = np.arange(T) % 4 != 3
        self.x = self.t.x
        self.layer = gpu_layer(device, self.t, training=training)
        self.layer.set_feed_forward_norm(self.norm, EPS)
        self.layer.set_block_join(self.post, self.gate, scale, EPS)
        self.layout = rb.Layout(valid=self.live.tolist() if padding else None)
        self.valid = self.live.astype(np.uint8) if padding else None

    def want(self):
        self.normed = self.stored(orc.rmsnorm(self.x, self.norm, EPS))
        self.y = oracle_layer(self.t).forward(self.normed, valid=self.valid).out
        wide = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
        return jo.forward(self.x.astype(np.float64), self.y.astype(np.float64), self.live, wide(self.post), wide(self.gate),
                          float(np.float32(self.scale)), EPS)


SHAPES = [dict(d=64, E=8, k=2, F=64, T=1), dict(d=128, E=8, k=2, F=64, T=5, shared=True), dict(d=64, E=4, k=2, F=64, T=300, shared=True),
          dict(d=33, E=5, k=2, F=19, T=65), dict(d=768, E=8, k=2, F=128, T=130)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "d{d}_T{T}".format(**s))
@pytest.mark.parametrize("act,wt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "int8"), ("f32", "bf16")])
@pytest.mark.parametrize("post,gate,scale", [(True, True, 0.4), (False, True, 1.0), (True, False, 1.0), (False, False, 0.22)])
def test_forward(device, shape, act, wt, post, gate, scale):
    b = Block(device, shape, act, wt, post, gate, scale, padding=shape["T"] > 4)
    want = b.want()
    out, _ = b.layer.forward_block(b.x, b.layout)
    tol = tolerance(b.t.workload)
    assert rel_l2(out, want) <= tol
    # the branch alone; a bf16 output carries the rounding of the sum
    share = float(np.linalg.norm(want - b.x))
    rounding = 2.0 ** -8 * float(np.linalg.norm(want)) / max(share, 1e-30) if b.bf16 else 0.0
    assert rel_l2(out - b.x, want - b.x) <= 2 * tol + rounding
    assert np.array_equal(out[~b.live], b.x[~b.live])
    b.layer.close()


@pytest.mark.parametrize("shape", SHAPES[1:], ids=lambda s: "d{d}_T{T}".format(**s))
@pytest.mark.parametrize("act,wt", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("post,gate,scale", [(True, True, 0.4), (False, False, 0.22), (True, False, 1.0)])
def test_backward(device, shape, act, wt, post, gate, scale):
    b = Block(device, shape, act, wt, post, gate, scale, training=True, padding=True)
    b.want()
    b.layer.zero_grads()
    gout = b.stored(np.random.default_rng(4).standard_normal(b.x.shape))
    b.layer.forward_block(b.x, b.layout)
    got = b.layer.backward_block(gout)
    wide = lambda v: None if v is None else v.astype(np.float64)  # noqa: E731
    g, _ = jo.backward(b.y.astype(np.float64), None, b.live, wide(b.post), wide(b.gate), float(np.float32(scale)), None, EPS,
                       gout.astype(np.float64), None, True)
    inner = oracle_layer(b.t).backward(b.normed, g["grad_y"].astype(np.float32), valid=b.valid)
    gi, gw = orc.rmsnorm_backward(b.x, inner.grad_input, b.norm, EPS)
    tol = 3e-5 if act == "f32" else 2e-2
    assert rel_l2(got, gi + gout) <= tol
    assert rel_l2(b.layer.weight_grad(L.W_NORM).reshape(-1), gw) <= tol
    assert rel_l2(b.layer.weight_grad(L.W_DOWN, 1), inner.grad_down[1]) <= tol
    if post:
        assert rel_l2(b.layer.weight_grad(L.W_POST_NORM).reshape(-1), g["grad_post"]) <= tol
    if gate:
        assert rel_l2(b.layer.weight_grad(L.W_BLOCK_GATE).reshape(-1), g["grad_gate"]) <= tol
        first = b.layer.weight_grad(L.W_BLOCK_GATE)
        b.layer.forward_block(b.x, b.layout)
        b.layer.backward_block(gout)
        assert rel_l2(b.layer.weight_grad(L.W_BLOCK_GATE), 2 * first) <= 1e-6   # gradients accumulate
        b.layer.zero_grads()
        assert (b.layer.weight_grad(L.W_BLOCK_GATE) == 0).all()
    b.layer.close()


def bits(b, a):
    return synth.f32_to_bf16_bits(a) if b.bf16 else np.ascontiguousarray(a, np.float32)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_the_block_and_the_operator_give_the_same_bits(device, act):
    b = Block(device, dict(d=128, E=8, k=2, F=64, T=300), act, act)
    b.want()
    y, _ = b.layer.forward_train(b.normed)
    up = lambda a: DeviceBuffer(device, a.nbytes).upload(a)  # noqa: E731
    x, yb, post, gate = up(bits(b, b.x)), up(bits(b, y)), up(b.post), up(b.gate)
    out = DeviceBuffer(device, x.nbytes)
    j = rb.ResidualJoin(device, 128, dtype=act, gate="channel")
    j.forward_device(300, x.ptr, yb.ptr, out.ptr, post_weight_ptr=post.ptr, gate_ptr=gate.ptr, scale=b.scale, eps=EPS)
    device.synchronize()
    alone = out.download(np.empty_like(bits(b, b.x)))
    b.layer.forward_block_device(x.ptr, 300, x.ptr)  # in place
    device.synchronize()
    assert np.array_equal(alone, x.download(np.empty_like(alone)))


def test_back_to_the_residual_add(device):
    b = Block(device, dict(d=128, E=8, k=2, F=64, T=40), "bf16", "bf16")
    joined, _ = b.layer.forward_block(b.x)
    b.layer.set_block_join()
    plain, _ = b.layer.forward_block(b.x)
    other = gpu_layer(device, b.t)
    other.set_feed_forward_norm(b.norm, EPS)
    want, _ = other.forward_block(b.x)
    assert np.array_equal(plain, want) and not np.array_equal(plain, joined)


def test_refusals(device):
    t = synth.make(small_workload(d=64, E=4, k=2, F=64, T=40, seed=5, act="bf16", wt="bf16"))
    layer = gpu_layer(device, t, training=True)
    w = np.ones(64, np.float32)
    with pytest.raises(rb.InvalidConfig, match="norm has not been set"):
        layer.set_block_join(w)
    layer.set_feed_forward_norm(w)
    for bad in (dict(post_weight=np.ones(63)), dict(gate=np.ones(65)), dict(scale=float("nan")), dict(eps=-1.0), dict(eps=float("inf"))):
        with pytest.raises(rb.InvalidInput):
            layer.set_block_join(**bad)
    for which in (L.W_POST_NORM, L.W_BLOCK_GATE):
        with pytest.raises(rb.InvalidConfig):
            layer.weight_grad(which)
    layer.forward_block(t.x)
    layer.set_block_join(w)
    with pytest.raises(rb.InvalidInput):  # the forward had no norm behind it
        layer.backward_block(t.x)
    layer.forward_block(t.x)
    layer.backward_block(t.x)
    with pytest.raises(rb.InvalidConfig):
        layer.weight_grad(L.W_BLOCK_GATE)
    assert layer.weight_grad(L.W_POST_NORM).shape == (1, 64)
    lib = L.load()
    assert lib.rbmoe_set_block_join(None, None, None, 64, 1e-6, 1.0) == L.NULL_POINTER


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_a_training_step_with_join_and_update_replays_like_the_eager_one(device, hip, act):  # noqa: F811
    """zero gradients, block step forward and backward, update: captured once, replayed with eager work in between, against a twin layer."""
    shape = dict(d=128, E=4, k=2, F=64, T=300, shared=True)
    t = synth.make(small_workload(seed=77, act=act, wt=act, **shape))
    rng = np.random.default_rng(3)
    norm, post, gate = (rng.uniform(0.5, 1.5, 128).astype(np.float32) for _ in range(3))

    def make():
        w = t.workload
        cfg = rb.MoeConfig(w.num_experts, w.experts_per_token, w.d_ff, True)
        layer = rb.MoeLayer(128, cfg, device, act_dtype=act, weight_dtype=act, max_tokens=300, shared_d_ff=w.shared_d_ff)
        layer.enable_training()
        layer.enable_muon()
        layer.load_tensors(t)
        layer.set_feed_forward_norm(norm)
        layer.set_block_join(post, gate, 0.5)
        return layer

    to_bits = (lambda a: synth.f32_to_bf16_bits(a)) if act == "bf16" else (lambda a: np.ascontiguousarray(a, np.float32))
    xh = to_bits(t.x)
    gh = to_bits(rng.standard_normal(t.x.shape).astype(np.float32))
    x, g = DeviceBuffer(device, xh.nbytes).upload(xh), DeviceBuffer(device, gh.nbytes).upload(gh)
    layers = [make(), make()]
    outs = [(DeviceBuffer(device, xh.nbytes), DeviceBuffer(device, xh.nbytes)) for _ in range(2)]

    def step(i):
        layers[i].zero_grads()
        layers[i].forward_block_device(x.ptr, 300, outs[i][0].ptr)
        layers[i].backward_block_device(g.ptr, 300, outs[i][1].ptr)
        layers[i].muon_step(0.02, weight_decay=0.1)

    cap = Capture(hip, device, lambda: step(1))
    for _ in range(4):
        device.set_stream(None)
        step(0)
        device.synchronize()
        cap.replay()
        device.synchronize()
        for a, b in zip(outs[0], outs[1]):
            assert np.array_equal(a.download(np.empty_like(xh)), b.download(np.empty_like(xh)))
        for which, e in ((L.W_GATE, 0), (L.W_DOWN, 3), (L.W_SHARED_UP, 0)):
            assert np.array_equal(layers[0].weight(which, e), layers[1].weight(which, e))
        assert np.array_equal(layers[0].weight_grad(L.W_POST_NORM), layers[1].weight_grad(L.W_POST_NORM))
    cap.close()
