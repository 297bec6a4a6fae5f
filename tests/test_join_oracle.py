"""The 64-bit gradients that the device's are held to, against differences of the forward formula.  No GPU."""
import ctypes as C

import numpy as np
import pytest

import join_oracle as jo
import rustingbrain_amd as rb
from rustingbrain_amd import _lib as L


@pytest.mark.parametrize("gate", ["none", "channel", "row"])
@pytest.mark.parametrize("post,following", [(True, True), (False, True), (True, False), (False, False)])
def test_gradients_against_differences(gate, post, following):
    rng = np.random.default_rng(3)
    r, d, scale, eps = 5, 7, 0.3, 1e-3
    live = np.array([True, True, False, True, True])
    v = {"x": rng.standard_normal((r, d)), "y": rng.standard_normal((r, d)), "post": 1 + 0.1 * rng.standard_normal(d) if post else None,
         "gate": None if gate == "none" else rng.standard_normal(d if gate == "channel" else (r, d)),
         "next": 1 + 0.1 * rng.standard_normal(d) if following else None}
    go, gn = rng.standard_normal((r, d)), rng.standard_normal((r, d)) if following else None

    def loss(a):
        out = jo.forward(a["x"], a["y"], live, a["post"], a["gate"], scale, eps)
        # (a padding row's normed row takes part in grad_x, and in no parameter's gradient: the parameter is held for it)
        t = (out * go).sum()
        if following:
            n = jo.rms_norm(out, eps)
            t += (n * np.where(live[:, None], a["next"], v["next"]) * gn).sum()
        return t

    out = jo.forward(v["x"], v["y"], live, v["post"], v["gate"], scale, eps)
    got, _ = jo.backward(v["y"], out, live, v["post"], v["gate"], scale, v["next"], eps, go, gn, gate == "channel")
    h = 1e-5
    for name, key in (("x", "grad_x"), ("y", "grad_y"), ("post", "grad_post"), ("gate", "grad_gate"), ("next", "grad_next")):
        if v[name] is None:
            continue
        for at in np.ndindex(v[name].shape):
            up, down = {**v, name: v[name].copy()}, {**v, name: v[name].copy()}
            up[name][at] += h
            down[name][at] -= h
            # central difference: h^2 / 6 times a third derivative of order 10, and 64-bit roundings over h
            assert abs((loss(up) - loss(down)) / (2 * h) - got[key][at]) < 1e-7, (name, at)


def test_calls_without_a_handle_are_refused():
    lib = L.load()
    h = C.c_void_p()
    assert lib.rbmoe_join_create(None, 8, L.F32, 0, C.byref(h)) == L.NULL_POINTER
    assert lib.rbmoe_join_forward(None, 1, None, None, None, None, None, 1.0, None, 1e-6, None, None) == L.NULL_POINTER
    assert lib.rbmoe_join_backward(None, 1, None, None, None, None, None, 1.0, None, 1e-6, None, None, 0, None, None, None, None,
                                   None) == L.NULL_POINTER
    assert lib.rbmoe_muon_create(None, 1, 8, 8, C.byref(h)) == L.NULL_POINTER
    assert lib.rbmoe_orthogonalize(None, None, L.F32, 5, None, L.F32) == L.NULL_POINTER
    assert lib.rbmoe_muon_step(None, None, L.F32, None, None, 0.1, 0.9, 0.0, 0.0, 1, 5) == L.NULL_POINTER
    lib.rbmoe_join_destroy(None)
    lib.rbmoe_muon_destroy(None)
    with pytest.raises(rb.InvalidConfig, match="gate"):
        rb.ResidualJoin(None, 8, gate="column")
