"""The accuracy that the kernels are held to (attention_precision) tells arithmetics apart: three parts of operands and six products pass, two parts and
three products, or fewer, do not; bf16 rows whose ds are not mended do not.  No GPU."""
import numpy as np
import pytest

import attention_oracle as ao
import attention_precision as ap


def problem(nq, nk, d):
    q, k, v, go = ap.rows(np.random.default_rng(nq + d), nq, nk, d)
    mask, scale = ao.seen(nq, nk, True), np.float32(d ** -0.5)
    want = ap.formulas(*(a.astype(np.float64) for a in (q, k, v, go)), mask, float(scale))
    return (q, k, v, go), mask, scale, want, ap.formulas(q, k, v, go, mask, scale)


def test_the_formulas_are_the_oracles():
    (q, k, v, go), mask, scale, want, _ = problem(70, 90, 40)
    other = ao.head(*(a.astype(np.float64) for a in (q, k, v)), mask, float(scale), "f32", go.astype(np.float64))
    for name in ap.NAMES:
        assert np.allclose(want[name], other[name][0], rtol=1e-12, atol=1e-12), name


@pytest.mark.parametrize("nq,nk,d", [(300, 300, 64), (1000, 1000, 64), (300, 300, 128), (130, 700, 40)])
def test_parts_of_operands(nq, nk, d):
    arrays, mask, scale, want, f32 = problem(nq, nk, d)
    wide = [a.astype(np.float64) for a in arrays]
    assert not ap.as_exact_as_f32(f32, f32, want)
    assert not ap.as_exact_as_f32(ap.formulas(*wide, mask, float(scale), ap.in_parts(3, 3)), f32, want)
    for parts, dropped in ((2, 2), (2, 3), (1, 1)):
        bad = ap.as_exact_as_f32(ap.formulas(*wide, mask, float(scale), ap.in_parts(parts, dropped)), f32, want)
        assert set(bad) == set(ap.NAMES), (parts, bad)


@pytest.mark.parametrize("nq,nk,d", [(300, 300, 64), (600, 600, 128), (130, 700, 40)])
def test_ds_that_do_not_add_up_to_nothing(nq, nk, d):
    q, k, v, go = (ap.rounded(a) for a in ap.rows(np.random.default_rng(nq + d), nq, nk, d))
    mask, scale = ao.seen(nq, nk, True), d ** -0.5
    want = ap.formulas(q, k, v, go, mask, scale)
    model, plain = (ap.bf16_rounded(q, k, v, go, mask, scale, mended) for mended in (True, False))
    got = {n: ap.rounded(a) for n, a in model.items()}
    assert not ap.as_exact_as_bf16(got, model, want)
    for name in ("out", "grad_q", "grad_k", "grad_v"):
        err, norm = ap.error(got[name], want[name])
        assert err <= 0.0027 * norm, (name, err / norm)  # (sqrt(2) roundings of the result, and what a few keys a row add)
    bad = ap.as_exact_as_bf16({n: ap.rounded(a) for n, a in plain.items()}, model, want)
    assert "grad_q" in bad, bad  # (keys share a direction, queries do not: grad_k hardly shows it)
