"""As many sequences as a call may have, of a row or none each: a row that sees one key has its value, and gradients that are known without a sum."""
import numpy as np
import pytest

import rustingbrain_amd as rb
from test_gpu_attention import Ints
from test_gpu_join import Array, stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads", [(2, 1, 8), (4, 4, 72)])
def test_most_sequences(device, dtype, heads):
    n, (h, kv, d) = 65535, heads
    rng = np.random.default_rng(h)
    counts = (rng.random(n) < 0.7).astype(np.int32)
    begin = np.concatenate([[0], np.cumsum(counts)[:-1]]).astype(np.int32)
    rows = int(counts.sum())
    q, k, v, go = (stored(rng.standard_normal((rows, x, d)), dtype) for x in (h, kv, kv, h))
    arrays = [Array(device, a.shape, dtype, a) for a in (q, k, v)]
    dgo, out, lse = Array(device, go.shape, dtype, go), Array(device, q.shape, dtype), Array(device, (h, rows), "f32")
    grads = [Array(device, a.shape, dtype) for a in (q, k, v)]
    b, c = Ints(device, begin), Ints(device, counts)
    op = rb.Attention(device, h, kv, d, dtype=dtype, backward_rows=rows)
    where = dict(query_begin_ptr=b.ptr, query_count_ptr=c.ptr, query_rows=rows, key_rows=rows, longest_queries=1, longest_keys=1)
    op.forward_device(n, *(a.ptr for a in arrays), out.ptr, lse_ptr=lse.ptr, **where)
    op.backward_device(n, *(a.ptr for a in arrays), out.ptr, lse.ptr, dgo.ptr, *(a.ptr for a in grads), **where)
    device.synchronize()
    assert np.array_equal(out.get(), np.repeat(v, h // kv, axis=1))
    assert not grads[0].get().any() and not grads[1].get().any()
    # (p = exp(s - lse): its argument is off by a few roundings of s, as are a result's)
    want = go.reshape(rows, kv, h // kv, d).astype(np.float64)
    size, score = np.abs(want).sum(axis=2), np.abs(q).max() * np.abs(k).max() * d ** 0.5
    u = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    assert (np.abs(grads[2].get() - want.sum(axis=2)) <= size * (2 * u + 8 * 2.0 ** -24 * (score + 4))).all()
    op.close()
