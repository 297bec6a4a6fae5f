"""Training mode switched on between a block step's forward and its backward."""
import numpy as np
import pytest

import rustingbrain_amd as rb
from helpers import small_workload
from rustingbrain_amd import _lib as L
from rustingbrain_amd import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 300])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("join", [False, True])
def test_a_block_step_from_before_training_mode_has_no_backward(device, act, T, join):
    """It keeps neither the rows in front of the norm nor which of them are padding."""
    t = synth.make(small_workload(d=64, E=4, k=2, F=64, T=T, seed=34, act=act, wt=act))
    rng = np.random.default_rng(1)
    norm, post, gate = (rng.uniform(0.5, 1.5, 64).astype(np.float32) for _ in range(3))
    layout = rb.Layout(valid=[i % 3 != 1 for i in range(T)])

    def make(training):
        layer = rb.MoeLayer(64, rb.MoeConfig(4, 2, 64), device, act_dtype=act, weight_dtype=act, max_tokens=T)
        if training:
            layer.enable_training()
        layer.set_feed_forward_norm(norm)
        if join:
            layer.set_block_join(post, gate, 0.5)
        return layer

    layer, fresh = make(False), make(True)
    layer.forward_block(t.x, layout)
    layer.enable_training()
    with pytest.raises(rb.InvalidInput, match="training mode"):
        layer.backward_block(t.x)
    assert (layer.weight_grad(L.W_NORM) == 0).all()
    if join:
        assert (layer.weight_grad(L.W_POST_NORM) == 0).all() and (layer.weight_grad(L.W_BLOCK_GATE) == 0).all()
    got = []
    for each in (layer, fresh):
        each.load_tensors(t)
        each.forward_block(t.x, layout)
        got.append([each.backward_block(t.x)] + [each.weight_grad(w) for w in (L.W_NORM, L.W_ROUTER, L.W_DOWN)] +
                   ([each.weight_grad(w) for w in (L.W_POST_NORM, L.W_BLOCK_GATE)] if join else []))
        each.close()
    assert all(np.array_equal(a, b) for a, b in zip(*got))
