"""Attention of whole sequences (``Attention``) against the same formulas in 64 bits, both ways; tolerances: attention_oracle."""
import numpy as np
import pytest

import attention_oracle as ao
import rustingbrain_amd as rb
from bench import DeviceBuffer
from rustingbrain_amd import synth
from test_gpu_join import Array, ptr, stored

pytestmark = pytest.mark.gpu


class Ints:
    def __init__(self, dev, values, dtype=np.int32):
        values = np.ascontiguousarray(values, dtype)
        self.buf = DeviceBuffer(dev, max(16, values.nbytes))
        if values.nbytes:
            self.buf.upload(np.concatenate([values.view(np.uint8).reshape(-1), np.zeros(max(0, 16 - values.nbytes), np.uint8)]))
        self.ptr = self.buf.ptr


def starts(counts, gap):
    """Where sequences of `counts` rows begin, `gap` rows of nothing in front of each and behind the last; and all rows."""
    at, got = gap, []
    for n in counts:
        got.append(at)
        at += n + gap
    return got, at


class Problem:
    """Sequences of `counts` queries and `counts` + `earlier` keys (negative: fewer keys than queries).  `fused`: q, k and v side by side in one array.
    Rows between the sequences hold NaN, as do the outputs' before a call."""

    def __init__(self, dev, counts, earlier, heads, dtype, causal=True, gap=0, shift=0, fused=False, scale=None, seed=0, backward=True, spread=1.0):
        self.dev, self.dtype, self.causal, self.counts = dev, dtype, causal, list(counts)
        self.h, self.kv, self.d = heads
        self.scale = scale or 1.0 / np.sqrt(self.d)
        earlier = [earlier] * len(self.counts) if np.isscalar(earlier) else list(earlier)
        self.key_counts = [max(0, n + e) for n, e in zip(self.counts, earlier)]
        self.begin, self.rows = starts(self.counts, gap)
        self.key_begin, self.key_rows = starts(self.key_counts, gap)
        self.same = not any(earlier)
        fused = fused and self.same
        rng = np.random.default_rng([seed, self.rows, self.d, self.h])
        x = lambda rows, heads, std=1.0: stored(std * rng.standard_normal((rows, heads, self.d)), dtype)  # noqa: E731
        # keys and values share a direction: what a row loses by rounding adds up along it
        self.q = x(self.rows, self.h, 1.3 * spread)
        self.k = stored(x(self.key_rows, self.kv) + 1.5 * rng.standard_normal((1, self.kv, self.d)), dtype)
        self.v = stored(x(self.key_rows, self.kv) + 0.5 * rng.standard_normal((1, self.kv, self.d)), dtype)
        self.go = x(self.rows, self.h, 0.1)
        for a, begin, counts in ((self.q, self.begin, self.counts), (self.go, self.begin, self.counts), (self.k, self.key_begin, self.key_counts),
                                 (self.v, self.key_begin, self.key_counts)):
            a[~self.inside(begin, counts, len(a))] = np.nan
        self.fused = fused
        if fused:
            self.stride = (self.h + 2 * self.kv) * self.d + 8
            pad = np.full((self.rows, 8), np.nan, np.float32)
            both = np.concatenate([a.reshape(self.rows, -1) for a in (self.q, self.k, self.v)] + [pad], axis=1)
            self.all = Array(dev, both.shape, dtype, both, shift)
            self.strides = dict(q_stride=self.stride, k_stride=self.stride, v_stride=self.stride)
        else:
            self.dq, self.dk, self.dv = (Array(dev, a.shape, dtype, a, shift) for a in (self.q, self.k, self.v))
            self.strides = {}
        self.dgo = Array(dev, self.go.shape, dtype, self.go, shift)
        self.shift = shift
        self.ints = [Ints(dev, v) for v in (self.begin, self.counts, self.key_begin, self.key_counts)]
        self.op = rb.Attention(dev, self.h, self.kv, self.d, dtype=dtype, backward_rows=self.rows if backward else 0)

    @staticmethod
    def inside(begin, counts, rows):
        live = np.zeros(rows, bool)
        for b, n in zip(begin, counts):
            live[b:b + n] = True
        return live

    def inputs(self):
        if not self.fused:
            return [ptr(a) for a in (self.dq, self.dk, self.dv)]
        es = 2 if self.dtype == "bf16" else 4
        return [self.all.ptr, self.all.ptr + self.h * self.d * es, self.all.ptr + (self.h + self.kv) * self.d * es]

    def where(self, **more):
        i = self.ints
        keys = {} if self.same else dict(key_begin_ptr=i[2].ptr, key_count_ptr=i[3].ptr)
        return {**dict(query_begin_ptr=i[0].ptr, query_count_ptr=i[1].ptr, query_rows=self.rows, key_rows=self.key_rows,
                       longest_queries=max(self.counts, default=0), longest_keys=max(self.key_counts, default=0), causal=self.causal, scale=self.scale),
                **keys, **self.strides, **more}

    def forward(self, **more):
        self.out = Array(self.dev, self.q.shape, self.dtype, None, self.shift)
        self.lse = Array(self.dev, (self.h, self.rows), "f32", None)
        self.op.forward_device(len(self.counts), *self.inputs(), self.out.ptr, lse_ptr=self.lse.ptr, **self.where(**more))
        self.dev.synchronize()
        return {"out": self.out.get(), "lse": self.lse.get()}

    def backward(self, **more):
        if self.fused:
            grads = Array(self.dev, self.all.shape, self.dtype, None, self.shift)
            es = 2 if self.dtype == "bf16" else 4
            at = [grads.ptr, grads.ptr + self.h * self.d * es, grads.ptr + (self.h + self.kv) * self.d * es]
        else:
            grads = [Array(self.dev, a.shape, self.dtype, None, self.shift) for a in (self.q, self.k, self.v)]
            at = [a.ptr for a in grads]
        self.op.backward_device(len(self.counts), *self.inputs(), self.out.ptr, self.lse.ptr, self.dgo.ptr, *at, **self.where(**more))
        self.dev.synchronize()
        if self.fused:
            g = grads.get()
            cut = [0, self.h * self.d, (self.h + self.kv) * self.d, (self.h + 2 * self.kv) * self.d]
            assert untouched(g[:, cut[3]:], self.dtype)
            return {n: g[:, a:b].reshape(self.rows, -1, self.d) for n, a, b in zip(("grad_q", "grad_k", "grad_v"), cut, cut[1:])}
        return dict(zip(("grad_q", "grad_k", "grad_v"), (a.get() for a in grads)))

    def wanted(self, backward=True):
        """{name: (value, bound)} over all rows; rows outside the sequences are NaN."""
        group = self.h // self.kv
        new = lambda shape: [np.full(shape, np.nan), np.full(shape, 0.0)]  # noqa: E731
        got = {"out": new(self.q.shape), "lse": new((self.h, self.rows))}
        if backward:
            got.update(grad_q=new(self.q.shape), grad_k=new(self.k.shape), grad_v=new(self.v.shape))
        for b, n, kb, m in zip(self.begin, self.counts, self.key_begin, self.key_counts):
            mask = ao.seen(n, m, self.causal)
            for name in ("grad_k", "grad_v") if backward else ():
                got[name][0][kb:kb + m] = 0.0
            for h in range(self.h):
                r = ao.head(*(a.astype(np.float64) for a in (self.q[b:b + n, h], self.k[kb:kb + m, h // group], self.v[kb:kb + m, h // group])),
                            mask, self.scale, self.dtype, self.go[b:b + n, h].astype(np.float64) if backward else None)
                for name, pair in r.items():
                    for i in range(2):
                        if name == "lse":
                            got[name][i][h, b:b + n] = pair[i]
                        elif name in ("grad_k", "grad_v"):
                            got[name][i][kb:kb + m, h // group] += pair[i]
                        else:
                            got[name][i][b:b + n, h] = pair[i]
        return got


def untouched(a, dtype):
    bits = synth.f32_to_bf16_bits(a) if dtype == "bf16" else np.ascontiguousarray(a).view(np.uint32)
    return bool((bits == (0xA5A5 if dtype == "bf16" else 0xA5A5A5A5)).all())


def check(got, want, dtype, what=""):
    for name, g in got.items():
        value, bound = want[name]
        outside = np.isnan(value)
        assert untouched(g[outside], "f32" if name == "lse" else dtype), f"{what} {name}: rows outside the sequences changed"
        g, value, bound = g[~outside].astype(np.float64), value[~outside], bound[~outside]
        with np.errstate(invalid="ignore"):
            bad = ~((np.abs(g - value) <= bound) | (g == value))
        assert not bad.any(), (what, name, int(bad.sum()), bad.size, np.argwhere(bad)[:3].tolist(), g[bad][:4], value[bad][:4], bound[bad][:4])


DEFAULT = (8, 2, 64)
CASES = [
    # counts, earlier, heads, causal, gap, shift, fused
    ([1], 0, DEFAULT, True, 0, 0, False),
    ([2, 1, 3], 0, (2, 1, 64), True, 0, 0, True),
    ([33], 0, (1, 1, 128), True, 0, 0, False),
    ([77, 130, 1, 64], 0, DEFAULT, True, 0, 0, True),
    ([128, 129, 127], 0, (4, 1, 128), True, 3, 0, False),
    ([300], 0, (2, 2, 32), True, 0, 0, False),
    ([200, 65], 0, (6, 3, 80), True, 1, 0, True),
    ([97], 0, (3, 1, 8), True, 0, 0, False),
    ([150, 40], 0, (5, 5, 40), True, 0, 1, False),       # rows off 16 bytes
    ([150, 31], 0, (4, 2, 104), True, 2, 3, True),
    ([70, 5], 0, (2, 1, 64), False, 0, 0, False),
    ([260], 0, (2, 1, 128), False, 0, 0, True),
    ([1, 1, 5], [200, 0, 131], (4, 2, 64), True, 0, 0, False),  # behind a cache
    ([40, 130], [300, 3], (4, 4, 128), True, 2, 0, False),
    ([40, 130], [300, 3], (2, 1, 48), False, 0, 1, False),
    ([100, 7, 200], [-60, -7, -128], (2, 1, 64), True, 1, 0, False),  # rows that see no key, a sequence without any
    ([50, 9], [-50, -3], (4, 2, 128), False, 0, 0, False),
    ([0, 60, 0], [0, 0, 30], (2, 1, 64), True, 0, 0, False),  # sequences without a row
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_and_backward(device, dtype, case):
    counts, earlier, heads, causal, gap, shift, fused = CASES[case]
    p = Problem(device, counts, earlier, heads, dtype, causal, gap, shift, fused, seed=case)
    want = p.wanted()
    check(p.forward(), want, dtype, "forward")
    check(p.backward(), want, dtype, "backward")
    p.op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [0.0, 8.0])
def test_flat_and_steep_rows(device, dtype, spread):
    """Every key alike, and a few keys for all: the running maximum moves far."""
    p = Problem(device, [300], 0, (2, 1, 64), dtype, spread=spread)
    if spread:
        p.k *= np.linspace(0.2, 1.0, 300).astype(np.float32)[:, None, None]
        p.k = stored(p.k, dtype)
        p.dk = Array(device, p.k.shape, dtype, p.k)
    want = p.wanted()
    check(p.forward(), want, dtype)
    check(p.backward(), want, dtype)
    p.op.close()
