"""The paged cache (``KvCache``) and the attention of new rows over it (``DecodeAttention``).

Rows come back as they went in, or in 8 bits as the rule says, bit for bit.  The attention is held against 64 bits over the rows that the cache
holds (attention_oracle); p goes into the second product as two (bf16 rows) or three (f32 rows over 8 bits) bf16 parts, which
keep 16 and 24 bits of it."""
import numpy as np
import pytest

import attention_oracle as ao
import rustingbrain_amd as rb
from rustingbrain_amd import synth
from test_gpu_attention import Ints, untouched
from test_gpu_join import Array, stored

pytestmark = pytest.mark.gpu
TYPES = [("bf16", "bf16"), ("bf16", "int8"), ("f32", "f32"), ("f32", "int8")]


def as_cached(x, dtype, cache):
    """What rows [.., d] are in the cache, as f32 values of the rows' type when they are read."""
    x = np.asarray(x, np.float32)
    if cache != "int8":
        return x, x
    with np.errstate(all="ignore"):
        most = np.abs(x).max(axis=-1, keepdims=True)
        scale = (most / np.float32(127)).astype(np.float32)
        small = np.where(most > 2.0 ** 100, np.float32(2.0 ** -20), np.float32(1))  # (127 x is in range, whatever x is)
        q = np.where(most > 0, np.rint((np.float32(127) * (x * small)).astype(np.float32) / (most * small)), np.float32(0)).astype(np.float32)
        kept = q * scale
    kept = np.where(np.isfinite(most), kept, np.float32(np.nan))
    return kept, stored(kept, dtype)


class Cache:
    """A cache with a copy of what it should hold."""

    def __init__(self, dev, kv, d, pages, page, dtype, cache):
        self.dev, self.kv, self.d, self.page, self.dtype, self.cache = dev, kv, d, page, dtype, cache
        self.op = rb.KvCache(dev, kv, d, pages, page_rows=page, dtype=dtype, cache_dtype=cache)
        self.kept = np.zeros((2, pages * page, kv, d), np.float32)  # keys, values

    def write(self, k, v, slots, shift=0, stride=0):
        slots = np.asarray(slots, np.int64)
        pad = lambda a: a if not stride else np.concatenate([a.reshape(len(a), -1), np.full((len(a), stride - self.kv * self.d), np.nan, np.float32)], axis=1)  # noqa: E731
        dk, dv = (Array(self.dev, pad(a).shape, self.dtype, pad(a), shift) for a in (k, v))
        s = Ints(self.dev, slots, np.int64)
        self.op.write_device(len(slots), dk.ptr, dv.ptr, s.ptr, k_stride=stride, v_stride=stride)
        self.dev.synchronize()
        there = (slots >= 0) & (slots < self.kept.shape[1])
        for i, a in enumerate((k, v)):
            self.kept[i, slots[there]] = as_cached(a, self.dtype, self.cache)[0][there]

    def read(self, slots, shift=0):
        slots = np.asarray(slots, np.int64)
        k, v = (Array(self.dev, (len(slots), self.kv, self.d), self.dtype, None, shift) for _ in range(2))
        s = Ints(self.dev, slots, np.int64)
        self.op.read_device(len(slots), k.ptr, v.ptr, s.ptr)
        self.dev.synchronize()
        return k.get(), v.get()

    def expected(self, slots):
        slots = np.asarray(slots, np.int64)
        there = (slots >= 0) & (slots < self.kept.shape[1])
        got = np.where(there[None, :, None, None], self.kept[:, np.where(there, slots, 0)], np.float32(0))
        return stored(got, self.dtype)


def rows_of(rng, n, kv, d, dtype):
    return stored(rng.standard_normal((n, kv, d)) * np.exp(rng.standard_normal((n, kv, 1))), dtype)


def same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32) + 0, np.asarray(b, np.float32).view(np.uint32) + 0) or np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("kv,d,page", [(2, 64, 16), (1, 128, 64), (3, 80, 32), (2, 40, 16), (1, 8, 4096), (2, 104, 128)])
def test_rows_come_back(device, dtype, cache, kv, d, page):
    rng = np.random.default_rng(d)
    pages = max(3, 320 // page)
    c = Cache(device, kv, d, pages, page, dtype, cache)
    size = pages * page
    everywhere = np.arange(-2, size + 2)
    assert same(np.stack(c.read(everywhere)), c.expected(everywhere))  # zeros at first
    writes = [
        rng.permutation(size)[:100],                                   # scattered
        np.arange(3, 3 + 85),                                          # a run off every alignment
        np.arange(0, 64),
        np.concatenate([np.arange(40, 23, -1), [-1, size, size + 7, -(1 << 40), 1 << 40], np.arange(41, 60)]),  # backwards, and without a place
        np.array([size - 1]),
        np.array([-1]),
    ]
    for i, slots in enumerate(writes):
        shift = i % 2
        c.write(rows_of(rng, len(slots), kv, d, dtype), rows_of(rng, len(slots), kv, d, dtype), slots, shift, stride=kv * d + 6 if i % 3 == 1 else 0)
        for order in (everywhere, rng.permutation(size)[:77], np.arange(5, 5 + 70)):
            assert same(np.stack(c.read(order, shift)), c.expected(order)), i
    c.op.close()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (40, 128)])
def test_many_rows_come_back(device, dtype, cache, d, page):
    """Calls of more workgroups than compute units, whose values go through LDS in pieces."""
    rng, kv, size = np.random.default_rng(d), 16, 1280
    c = Cache(device, kv, d, size // page, page, dtype, cache)
    gaps = np.arange(1200)  # runs of every length, off every alignment, with rows of no place between
    gaps[rng.integers(0, 1200, 150)] = -1
    swapped = np.arange(1280).reshape(-1, 5)[:, ::-1].reshape(-1)
    for i, slots in enumerate((np.arange(7, 7 + 1270), gaps + np.where(gaps < 0, 0, 3), rng.permutation(size)[:1100], swapped)):
        c.write(rows_of(rng, len(slots), kv, d, dtype), rows_of(rng, len(slots), kv, d, dtype), slots, i % 2)
        for order in (np.arange(-1, size + 1), rng.permutation(size), slots):
            assert same(np.stack(c.read(order, i % 2)), c.expected(order)), i
    c.op.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_eight_bits_of_odd_rows(device, dtype):
    """Zeros, ties, one large value, values near the ends of the range, infinities and NaN; a row's scale is its own."""
    d = 64
    x = np.zeros((9, 1, d), np.float32)
    x[1, 0, :] = 1.0
    x[2, 0, :5] = [127.0, 0.5, 1.5, 2.5, -0.5]     # ties to even
    x[3, 0, :3] = [1.0, 0.5, -0.5]                 # 63.5
    x[4, 0, 7] = -3e38
    x[5, 0, :2] = [1e-30, -3e-33]
    x[6, 0, 3] = np.inf
    x[7, 0, 5], x[7, 0, 6] = np.nan, 2.0
    x[8, 0, 0], x[8, 0, 1] = -np.inf, np.nan
    x = stored(x, dtype)
    c = Cache(device, 1, d, 2, 16, dtype, "int8")
    c.write(x, x[::-1], np.arange(9))
    k, v = c.read(np.arange(16))
    assert same(np.stack([k, v]), c.expected(np.arange(16)))
    assert np.isnan(k[6:9]).all() and np.isfinite(k[:6]).all() and (k[9:] == 0).all()
    assert k[3, 0, 1] == stored(np.float32(64) * np.float32(1 / np.float32(127)), dtype)
    c.op.close()


class Sequences:
    """Sequences of `lengths` rows in pages handed out in a random order."""

    def __init__(self, dev, lengths, heads, page, dtype, cache, seed=0, free=2, extra_pages=0, spread=1.0):
        self.dev, self.dtype, self.lengths = dev, dtype, np.asarray(lengths, np.int32)
        self.h, self.kv, self.d = heads
        rng = np.random.default_rng([seed, int(self.lengths.sum()), self.d])
        need = [-(-int(n) // page) for n in self.lengths]
        pages = sum(need) + free
        order = list(rng.permutation(pages))
        self.table_pages = max(need, default=0) + extra_pages
        self.tables = np.full((len(need), self.table_pages), -7, np.int32)  # (entries behind a sequence's pages are not read)
        for i, n in enumerate(need):
            self.tables[i, :n] = [order.pop() for _ in range(n)]
        self.c = Cache(dev, self.kv, self.d, pages, page, dtype, cache)
        # what lies in the pages beside the sequences: values that would show
        junk = stored(np.full((pages * page, self.kv, self.d), np.nan, np.float32), dtype)
        self.c.write(junk, junk, np.arange(pages * page))
        for i, n in enumerate(self.lengths):
            at = np.arange(n)
            k = stored(rows_of(rng, n, self.kv, self.d, "f32") + rng.standard_normal((1, self.kv, self.d)), dtype)
            if n:
                self.c.write(k, rows_of(rng, n, self.kv, self.d, dtype), self.tables[i, at // page].astype(np.int64) * page + at % page)
        self.q = stored(spread * rng.standard_normal((len(need), self.h, self.d)), dtype)
        self.op = rb.DecodeAttention(dev, self.h, self.kv, self.d, max(1, len(need)), dtype=dtype)
        self.page = page

    def run(self, longest=None, shift=0, stride=0, scale=0.0):
        n = len(self.lengths)
        q = self.q.reshape(n, -1)
        if stride:
            q = np.concatenate([q, np.full((n, stride - q.shape[1]), np.nan, np.float32)], axis=1)
        dq, out = Array(self.dev, q.shape, self.dtype, q, shift), Array(self.dev, self.q.shape, self.dtype, None, shift)
        t, l = Ints(self.dev, self.tables), Ints(self.dev, self.lengths)
        self.op.forward_device(self.c.op, n, dq.ptr, out.ptr, t.ptr, self.table_pages, l.ptr, longest=max(self.lengths) if longest is None else longest,
                               q_stride=stride, scale=scale)
        self.dev.synchronize()
        return out.get()

    def check(self, got, lengths=None, tables=None, scale=None):
        lengths, tables = self.lengths if lengths is None else lengths, self.tables if tables is None else tables
        group = self.h // self.kv
        up = 2.0 ** -16 if self.dtype == "bf16" else 2.0 ** -23
        for i, n in enumerate(lengths):
            at = np.arange(max(0, n))
            pages = tables[i, at // self.page].astype(np.int64)
            live = (pages >= 0) & (pages < self.c.kept.shape[1] // self.page)
            slots = (pages * self.page + at % self.page)[live]
            for h in range(self.h):
                k, v = (self.c.kept[j, slots, h // group].astype(np.float64) for j in range(2))
                want, bound = ao.head(self.q[i, h][None].astype(np.float64), k, v, np.ones((1, len(slots)), bool), scale or self.d ** -0.5,
                                      self.dtype, up=up)["out"]
                bad = ~(np.abs(got[i, h] - want[0]) <= bound[0])
                assert not bad.any(), (i, h, int(bad.sum()), got[i, h][bad][:3], want[0][bad][:3], bound[0][bad][:3])


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("lengths,heads,page", [
    ([1], (8, 2, 64), 16), ([777], (8, 2, 64), 16), ([64, 1, 65, 63, 2, 128, 15, 16, 17], (4, 1, 128), 16),
    ([300, 0, 31], (6, 3, 80), 32), ([100, 513], (5, 5, 40), 128), ([2000, 3, 1111], (2, 2, 64), 64), ([50, 200], (40, 2, 128), 16),
    ([260], (17, 1, 8), 4096), ([33, 47], (16, 1, 104), 16)])
def test_decode(device, dtype, cache, lengths, heads, page):
    s = Sequences(device, lengths, heads, page, dtype, cache)
    s.check(s.run())
    s.check(s.run(longest=5000, shift=1, stride=heads[0] * heads[2] + 10))  # a launch for more than there is, rows off 16 bytes
    s.op.close()
    s.c.op.close()
