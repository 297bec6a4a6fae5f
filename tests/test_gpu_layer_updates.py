"""Updates of a layer's expert matrices on the device (``MoeLayer.enable_muon``, ``muon_step``, ``weight``): every matrix against the
same step in 64 bits (tolerance: test_gpu_muon), and the layer behind it against a fresh one that was given the updated weights, bit for
bit, forward and backward: that is what the stored operand order and the transposed copies are worth."""
import numpy as np
import pytest

import rustingbrain_amd as rb
from helpers import small_workload
from rustingbrain_amd import _lib as L
from rustingbrain_amd import synth
from test_gpu_muon import step

pytestmark = pytest.mark.gpu


def make(device, t, muon=True, training=True, load=True):
    w = t.workload
    cfg = rb.MoeConfig(w.num_experts, w.experts_per_token, w.d_ff, w.shared_expert)
    layer = rb.MoeLayer(w.d_model, cfg, device, act_dtype=w.act_dtype, weight_dtype=w.weight_dtype, max_tokens=t.x.shape[0],
                        shared_d_ff=w.shared_d_ff if w.shared_expert else 0)
    if training:
        layer.enable_training()
    if muon:
        layer.enable_muon()
    if load:
        layer.load_tensors(t)
    return layer


def matrices(w):
    out = [(which, e) for e in range(w.num_experts) for which in (L.W_GATE, L.W_UP, L.W_DOWN)]
    return out + ([(which, 0) for which in (L.W_SHARED_GATE, L.W_SHARED_UP, L.W_SHARED_DOWN)] if w.shared_expert else [])


CASES = [dict(d=128, E=4, k=2, F=64, T=100, act="bf16", wt="bf16", shared=True, shared_d_ff=128),   # whole tiles
         dict(d=64, E=5, k=2, F=40, T=70, act="bf16", wt="bf16", shared=True, shared_d_ff=72),        # widths rounded up to 64 and 128
         dict(d=72, E=3, k=1, F=50, T=40, act="bf16", wt="bf16"),                                    # any-shape kernels, plain bf16
         dict(d=64, E=4, k=2, F=48, T=90, act="f32", wt="f32", shared=True),                         # f32 rounded to 64
         dict(d=33, E=3, k=2, F=19, T=50, act="f32", wt="f32", shared=True),                         # f32 as they are
         dict(d=128, E=4, k=2, F=64, T=80, act="f32", wt="bf16"),                                    # f32 rows over bf16 weights
         dict(d=96, E=3, k=2, F=50, T=60, act="f32", wt="bf16", shared=True)]


@pytest.mark.parametrize("shape", CASES, ids=lambda s: "{act}_{wt}_d{d}_F{F}".format(**s))
def test_steps(device, shape):
    t = synth.make(small_workload(seed=91, **shape))
    layer = make(device, t)
    lr, mu, decay = 0.02, 0.9, 0.05
    f = lambda v: float(np.float32(v))  # noqa: E731
    weights = {m: layer.weight(*m) for m in matrices(t.workload)}
    for which, e in weights:  # what was given, not what is stored
        src = t.experts[e] if which < L.W_SHARED_GATE else t.shared
        given = src[{L.W_GATE: "gate", L.W_UP: "up", L.W_DOWN: "down", L.W_SHARED_GATE: "gate", L.W_SHARED_UP: "up", L.W_SHARED_DOWN: "down"}[which]]
        assert np.array_equal(weights[which, e], given)
    momentum = {m: np.zeros(w.shape) for m, w in weights.items()}
    rng = np.random.default_rng(2)
    for k in range(2):
        gout = rng.standard_normal(t.x.shape).astype(np.float32)
        gout = synth.round_bf16(gout) if shape["act"] == "bf16" else gout
        layer.zero_grads()
        layer.forward_train(t.x)
        layer.backward(gout)
        grads = {m: layer.weight_grad(*m) for m in weights}
        layer.muon_step(lr, momentum=mu, weight_decay=decay)
        for m, w in weights.items():
            rows, cols = w.shape
            scale = np.sqrt(max(1.0, rows / cols))
            want, wm, bound = step(w.astype(np.float64), momentum[m], grads[m].astype(np.float64), f(lr), f(mu), f(decay), scale, True)
            got = layer.weight(*m)
            # (the momentum is the device's f32 one: 2^-22 of it in front of the products, well inside their own bound)
            err = np.linalg.norm(got - want)
            assert err <= 1.5 * bound + 2.0 ** -22 * np.linalg.norm(want) + 2.0 ** -22 * lr * scale * np.sqrt(min(rows, cols)) * 1.21, (m, k, err, bound)
            assert np.array_equal(layer.weight_grad(*m), grads[m])
            momentum[m], weights[m] = wm, got
    fresh = make(device, t, muon=False, load=False)
    fresh.set_router(t.router)
    for e in range(t.workload.num_experts):
        fresh.set_expert(e, *(weights[which, e] for which in (L.W_GATE, L.W_UP, L.W_DOWN)))
    if t.shared is not None:
        fresh.set_shared(*(weights[which, 0] for which in (L.W_SHARED_GATE, L.W_SHARED_UP, L.W_SHARED_DOWN)))
    a, _ = layer.forward_train(t.x)
    b, _ = fresh.forward_train(t.x)
    assert np.array_equal(a, b)
    assert np.array_equal(layer.backward(gout), fresh.backward(gout))
    layer.close()
    fresh.close()


def test_weights_set_later_are_what_the_next_step_starts_from(device):
    t = synth.make(small_workload(d=64, E=2, k=1, F=64, T=40, seed=6, act="bf16", wt="bf16"))
    layer = make(device, t)
    new = [np.random.default_rng(i).standard_normal(s).astype(np.float32) for i, s in enumerate(((64, 64),) * 3)]
    layer.set_expert(1, *new)
    for which, w in zip((L.W_GATE, L.W_UP, L.W_DOWN), new):
        assert np.array_equal(layer.weight(which, 1), w)  # f32, though the stored weight is bf16


def test_refusals(device):
    t = synth.make(small_workload(d=64, E=2, k=1, F=64, T=40, seed=6, act="bf16", wt="bf16"))
    layer = make(device, t, muon=False, training=False, load=False)
    with pytest.raises(rb.InvalidConfig, match="training"):
        layer.enable_muon()
    layer.enable_training()
    with pytest.raises(rb.InvalidConfig, match="not enabled"):
        layer.muon_step(0.1)
    layer.load_tensors(t)
    with pytest.raises(rb.InvalidConfig, match="before the weights"):
        layer.enable_muon()
    with pytest.raises(rb.Unsupported):
        layer.weight(L.W_GATE, 0)
    layer = make(device, t)
    with pytest.raises(rb.InvalidInput, match="cleared"):
        layer.muon_step(0.1)
    layer.forward_train(t.x)
    layer.backward(t.x)
    for bad in (dict(lr=float("nan")), dict(lr=0.1, momentum=1.0), dict(lr=0.1, weight_decay=-0.1), dict(lr=0.1, update_scale=-1.0),
                dict(lr=0.1, steps=0)):
        with pytest.raises(rb.InvalidConfig):
            layer.muon_step(**bad)
    before = layer.weight(L.W_UP, 1)
    assert np.array_equal(before, t.experts[1]["up"])
    for bad in ((L.W_GATE, 2), (L.W_GATE, -1), (L.W_SHARED_UP, 0), (L.W_ROUTER, 0), (L.W_NORM, 0)):
        with pytest.raises(rb.InvalidConfig):
            layer.weight(*bad)
    layer.zero_grads()
    with pytest.raises(rb.InvalidInput):
        layer.muon_step(0.1)
    q = synth.make(small_workload(d=64, E=2, k=1, F=64, T=8, seed=6, act="bf16", wt="int8"))
    with pytest.raises(rb.InvalidConfig):
        make(device, q, training=False, load=False)
    f = synth.make(small_workload(d=64, E=2, k=1, F=64, T=8, seed=6, act="f32", wt="f32"))
    assert np.array_equal(make(device, f, muon=False, training=False).weight(L.W_DOWN, 1), f.experts[1]["down"])  # f32 layers hold them anyway
