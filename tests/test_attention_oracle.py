"""The oracle's gradients against differences of its forward, and its rows without a key.  No GPU."""
import numpy as np
import pytest

import attention_oracle as ao


@pytest.mark.parametrize("nq,nk,causal", [(5, 5, True), (7, 4, True), (3, 9, True), (4, 6, False)])
def test_gradients_are_those_of_the_forward(nq, nk, causal):
    rng = np.random.default_rng(nq)
    q, go = rng.standard_normal((2, nq, 8))
    k, v = rng.standard_normal((2, nk, 8))
    mask = ao.seen(nq, nk, causal)

    def loss(q, k, v):
        return (ao.head(q, k, v, mask, 0.3, "f32")["out"][0] * go).sum()

    got = ao.head(q, k, v, mask, 0.3, "f32", go)
    for i, name in enumerate(("grad_q", "grad_k", "grad_v")):
        args = [q, k, v]
        for at in np.ndindex(args[i].shape):
            h, x = 1e-6, args[i].copy()
            x[at] += h
            up = loss(*[x if j == i else a for j, a in enumerate(args)])
            x[at] -= 2 * h
            down = loss(*[x if j == i else a for j, a in enumerate(args)])
            assert abs((up - down) / (2 * h) - got[name][0][at]) < 1e-8, (name, at)


def test_rows_without_a_key():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((6, 8)), *rng.standard_normal((2, 2, 8))
    got = ao.head(q, k, v, ao.seen(6, 2, True), 0.3, "f32", rng.standard_normal((6, 8)))
    assert (got["out"][0][:4] == 0).all() and (got["lse"][0][:4] == -np.inf).all() and (got["grad_q"][0][:4] == 0).all()
    assert np.isfinite(got["lse"][0][4:]).all() and np.allclose(got["out"][0][4], v[0])
