"""How exact attention is: f32 rows beside the same formulas in f32, bf16 rows beside what rounding p, ds and the results costs, short
sequences of them beside what rounding the results alone costs (attention_precision has the tolerances)."""
import numpy as np
import pytest

import attention_oracle as ao
import attention_precision as ap
from test_gpu_attention import Problem

pytestmark = pytest.mark.gpu


def per_head(p, *arithmetics):
    """What each of [(type, formulas)] gives, laid out like the kernels'; the gradients of a kv head are summed over its group in that type."""
    group, scale = p.h // p.kv, np.float32(p.scale)
    got = []
    for kind, formulas in arithmetics:
        r = {"out": np.zeros(p.q.shape, kind), "lse": np.zeros((p.h, p.rows), kind), "grad_q": np.zeros(p.q.shape, kind),
             "grad_k": np.zeros(p.k.shape, kind), "grad_v": np.zeros(p.v.shape, kind)}
        for b, n, kb, m in zip(p.begin, p.counts, p.key_begin, p.key_counts):
            mask = ao.seen(n, m, p.causal)
            for h in range(p.h):
                f = formulas(*(a.astype(kind) for a in (p.q[b:b + n, h], p.k[kb:kb + m, h // group], p.v[kb:kb + m, h // group], p.go[b:b + n, h])), mask,
                             kind(scale))
                r["out"][b:b + n, h], r["lse"][h, b:b + n], r["grad_q"][b:b + n, h] = f["out"], f["lse"], f["grad_q"]
                r["grad_k"][kb:kb + m, h // group] += f["grad_k"]
                r["grad_v"][kb:kb + m, h // group] += f["grad_v"]
        got.append(r)
    return got


CASES = [
    ([300], 0, (2, 1, 64), True), ([1500], 0, (1, 1, 64), True), ([77, 200, 1], 0, (8, 2, 64), True), ([1100], 0, (2, 1, 128), True),
    ([33], 2000, (2, 2, 128), True), ([20, 40], [900, 1500], (4, 2, 64), True), ([300, 65], 0, (3, 3, 40), False), ([260], 0, (2, 2, 80), True),
    ([130] * 40, 0, (16, 8, 64), True), ([150] * 30, 0, (16, 16, 104), True)]


@pytest.mark.parametrize("counts,earlier,heads,causal", CASES)
def test_f32_rows_are_as_exact_as_f32(device, counts, earlier, heads, causal):
    p = Problem(device, counts, earlier, heads, "f32", causal)
    f32, want = per_head(p, (np.float32, ap.formulas), (np.float64, ap.formulas))
    got = {**p.forward(), **p.backward()}
    assert not ap.as_exact_as_f32(got, f32, want)
    p.op.close()


@pytest.mark.parametrize("counts,earlier,heads,causal", [
    ([1] * 30, 0, (4, 4, 64), True), ([2], 0, (8, 8, 64), True), ([2] * 10, 0, (6, 3, 80), False), ([2] * 24, 0, (24, 2, 128), True), ([4] * 24, 0, (6, 3, 80), True),
    ([1, 2, 3, 5, 9, 17], 0, (8, 2, 64), True), ([8] * 24, 0, (32, 4, 64), True), ([1, 2, 1], [3, 0, 9], (8, 8, 40), True)])
def test_short_f32_sequences_are_as_exact_as_f32(device, counts, earlier, heads, causal):
    """Where a key has most of a row's weight the formula in f32 rounds its score as it rounds lse, and p is nearly exact."""
    p = Problem(device, counts, earlier, heads, "f32", causal)
    f32, want = per_head(p, (np.float32, ap.formulas), (np.float64, ap.formulas))
    got = {**p.forward(), **p.backward()}
    assert not ap.as_exact_as_f32(got, f32, want)
    p.op.close()


@pytest.mark.parametrize("counts,earlier,heads,causal", CASES)
def test_bf16_rows_lose_what_rounding_costs(device, counts, earlier, heads, causal):
    p = Problem(device, counts, earlier, heads, "bf16", causal)
    model, want = per_head(p, (np.float64, ap.bf16_rounded), (np.float64, ap.formulas))
    got = {**p.forward(), **p.backward()}
    assert not ap.as_exact_as_bf16(got, model, want)
    p.op.close()


@pytest.mark.parametrize("counts,earlier,heads,causal", [
    ([1, 2, 3, 5, 32, 17], 0, (8, 2, 64), True), ([2], 0, (32, 4, 64), True), ([2, 2], 0, (8, 8, 64), False), ([2], 0, (24, 2, 128), True), ([2, 3], [160, 300], (5, 5, 40), True),
    ([300, 90], [-290, -70], (4, 2, 64), False), ([2, 30, 7] * 30, 0, (16, 16, 104), True), ([3] * 70, 40, (16, 8, 64), True)])
def test_gradients_of_short_bf16_sequences_are_rounded_once(device, counts, earlier, heads, causal):
    """p and ds have 16 bits there, 2^8 times as many as a result: what is left is the rounding of the result, but for values within a hundredth of a
    step of a tie."""
    p = Problem(device, counts, earlier, heads, "bf16", causal)
    want, = per_head(p, (np.float64, ap.formulas))
    p.forward()
    bad = ap.as_exact_as_f32(p.backward(), {n: ap.rounded(a) for n, a in want.items()}, want, 1.05, 2.0 ** -17)
    assert not bad
    p.op.close()
