"""Sequences that lie partly outside the arrays (``Attention``), both ways: the rows and keys that are there, each row with the keys that it would see if
all were there, and no row of another sequence; tolerances: attention_oracle."""
import numpy as np
import pytest

import attention_oracle as ao
import rustingbrain_amd as rb
from test_gpu_attention import Ints, Problem, check
from test_gpu_join import Array

pytestmark = pytest.mark.gpu


def wanted(p, sequences, causal):
    """{name: (value, bound)} of rows that stand alone or in sequences (query begin, count, key begin, count)."""
    new = lambda shape: [np.full(shape, np.nan), np.zeros(shape)]  # noqa: E731
    got = {"out": new(p.q.shape), "lse": new((p.h, p.rows)), "grad_q": new(p.q.shape), "grad_k": new(p.k.shape), "grad_v": new(p.v.shape)}
    group = p.h // p.kv
    for qb, nq, kb, nk in sequences:
        i, j = np.arange(nq), np.arange(nk)
        mask = (j[None] <= i[:, None] + nk - nq) if causal else np.ones((nq, nk), bool)
        i, j = i[(qb + i >= 0) & (qb + i < p.rows)], j[(kb + j >= 0) & (kb + j < p.key_rows)]
        rows, keys, mask = qb + i, kb + j, mask[np.ix_(i, j)]
        for name in ("grad_k", "grad_v"):
            got[name][0][keys] = 0.0
        for h in range(p.h):
            r = ao.head(*(a.astype(np.float64) for a in (p.q[rows, h], p.k[keys, h // group], p.v[keys, h // group])), mask, p.scale, p.dtype,
                        p.go[rows, h].astype(np.float64))
            for name, pair in r.items():
                for n in range(2):
                    if name == "lse":
                        got[name][n][h, rows] = pair[n]
                    elif name in ("grad_k", "grad_v"):
                        got[name][n][keys, h // group] += pair[n]
                    else:
                        got[name][n][rows, h] = pair[n]
    return got


def run(p, sequences, causal, **where):
    ints = [Ints(p.dev, [s[i] for s in sequences]) for i in range(4)]
    out, lse = Array(p.dev, p.q.shape, p.dtype), Array(p.dev, (p.h, p.rows), "f32")
    grads = [Array(p.dev, a.shape, p.dtype) for a in (p.q, p.k, p.v)]
    where = dict(dict(query_begin_ptr=ints[0].ptr, query_count_ptr=ints[1].ptr, key_begin_ptr=ints[2].ptr, key_count_ptr=ints[3].ptr, query_rows=p.rows,
                      key_rows=p.key_rows, longest_queries=max(s[1] for s in sequences), longest_keys=max(s[3] for s in sequences), causal=causal,
                      scale=p.scale), **where)
    n = len(sequences)
    p.op.forward_device(n, *p.inputs(), out.ptr, lse_ptr=lse.ptr, **where)
    p.op.backward_device(n, *p.inputs(), out.ptr, lse.ptr, p.dgo.ptr, *(g.ptr for g in grads), **where)
    p.dev.synchronize()
    return {"out": out.get(), "lse": lse.get(), **dict(zip(("grad_q", "grad_k", "grad_v"), (g.get() for g in grads)))}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(4, 2, 64), (16, 16, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_sequences_partly_outside(device, dtype, heads, causal):
    p = Problem(device, [150], 40, heads, dtype, causal)  # 150 rows, 190 keys
    cases = [
        # rows 0 .. 4 are the last of a sequence of ten; rows 5 .. 34 are another's
        [(-5, 10, -5, 10), (5, 30, 5, 30), (35, 200, 35, 200)],
        # rows behind their array, keys behind theirs, keys in front of theirs, a sequence whose rows are all outside
        [(100, 80, 60, 80), (0, 30, 170, 30), (30, 60, -20, 70), (-70, 60, 140, 20), (95, 0, 160, 5)],
    ]
    for sequences in cases:
        got = run(p, sequences, causal)
        check(got, wanted(p, sequences, causal), dtype, sequences)
    p.op.close()


def test_keys_beyond_an_array_of_fewer_rows(device):
    """One set of begins and counts for both, and fewer rows of keys than of queries: rows behind the last key see all that are left."""
    p = Problem(device, [120], -50, (4, 4, 64), "bf16")
    sequences = [(0, 40, 0, 40), (40, 80, 40, 80)]
    check(run(p, sequences, True, key_begin_ptr=0, key_count_ptr=0), wanted(p, sequences, True), "bf16")
    p.op.close()
