"""The attention operators called the ways a program calls them: prompts, cache and new rows together, captured and replayed, on a stream of the
caller's own, with sequences and tables that name places outside the arrays, with infinities and NaN in places that are not seen, over arrays whose
offsets pass 32 bits, and refused."""
import ctypes as C

import numpy as np
import pytest

import attention_oracle as ao
import rustingbrain_amd as rb
from bench import DeviceBuffer
from rustingbrain_amd import synth
from test_gpu_attention import Ints, Problem, check, untouched
from test_gpu_graph import Capture, hip  # noqa: F401  (a fixture)
from test_gpu_join import Array, stored
from test_gpu_kv_cache import Cache, Sequences, rows_of

pytestmark = pytest.mark.gpu


# ---- many workgroups: the waves of a workgroup share their tiles, where the small calls of test_gpu_attention have tiles a wave ----------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,causal,earlier,gap,shift", [
    ((16, 8, 64), True, 0, 0, 0), ((16, 16, 128), True, 0, 1, 0), ((24, 12, 40), False, 0, 0, 1), ((16, 8, 64), True, 70, 0, 0),
    ((12, 12, 104), True, -40, 2, 3)])
def test_many_workgroups(device, dtype, heads, causal, earlier, gap, shift):
    rng = np.random.default_rng(heads[0])
    counts = [1, 140, 128, 129, 64, 0] + list(rng.integers(1, 131, 34))
    p = Problem(device, counts, earlier, heads, dtype, causal, gap, shift, fused=not earlier and not gap)
    # (sequences * heads * tiles of 128 rows: over a thousand, of keys over five hundred)
    assert len(counts) * heads[1] * 2 >= 512
    want = p.wanted()
    check(p.forward(), want, dtype, "forward")
    check(p.backward(), want, dtype, "backward")
    p.op.close()


# ---- together -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "int8"), ("f32", "int8")])
def test_prompts_then_a_continued_prompt_then_new_rows(device, dtype, cache):
    """Three conversations through one layer's attention: prompts, written to the cache; more rows for two of them, whose earlier keys are read back
    from it; then new rows one by one.  Every output is that of the whole conversation so far over what the cache holds."""
    h, kv, d, page = 8, 2, 64, 16
    builder = rb.TransformerBuilder().max_seq_len(160)
    prompt = builder.build_attention(device, dtype=dtype)
    caches = builder.build_caches(device, sequences=3, dtype=dtype, cache_dtype=cache, page_rows=page)
    assert len(caches) == 8 and caches[0].pages == 30
    for c in caches[1:]:
        c.close()
    decode = builder.build_decode_attention(device, max_sequences=3, dtype=dtype)
    c = Cache(device, kv, d, 30, page, dtype, cache)
    c.op.close()
    c.op = caches[0]
    rng = np.random.default_rng(5)
    tables = rng.permutation(30).reshape(3, 10).astype(np.int32)
    slot = lambda i, at: tables[i, at // page].astype(np.int64) * page + at % page  # noqa: E731
    x = [[rows_of(rng, 160, n, d, dtype) for n in (h, kv, kv)] for _ in range(3)]
    have = [0, 0, 0]

    def held(i, n):  # what the cache holds of conversation i
        return c.kept[:, slot(i, np.arange(n))].astype(np.float64)

    def turn(more):
        """`more`[i] new rows of each conversation in one packed call."""
        who = [i for i in range(3) if more[i]]
        counts, keys = [more[i] for i in who], [have[i] + more[i] for i in who]
        q, k, v = (np.concatenate([x[i][j][have[i]:have[i] + more[i]] for i in who]) for j in range(3))
        slots = np.concatenate([slot(i, np.arange(have[i], have[i] + more[i])) for i in who])
        c.write(k, v, slots)
        # earlier rows come back from the cache, in 8 bits as they were rounded; the new ones too
        every = np.concatenate([slot(i, np.arange(n)) for i, n in zip(who, keys)])
        n = len(every)
        dk, dv = (Array(device, (n, kv, d), dtype) for _ in range(2))
        s = Ints(device, every, np.int64)
        caches[0].read_device(n, dk.ptr, dv.ptr, s.ptr)
        dq, out = Array(device, q.shape, dtype, q), Array(device, q.shape, dtype)
        at = lambda c: np.concatenate([[0], np.cumsum(c)[:-1]])  # noqa: E731
        ints = [Ints(device, a) for a in (at(counts), counts, at(keys), keys)]
        prompt.forward_device(len(who), dq.ptr, dk.ptr, dv.ptr, out.ptr, query_begin_ptr=ints[0].ptr, query_count_ptr=ints[1].ptr,
                              key_begin_ptr=ints[2].ptr, key_count_ptr=ints[3].ptr, query_rows=len(q), key_rows=n, longest_queries=max(counts),
                              longest_keys=max(keys))
        device.synchronize()
        got, first = out.get(), 0
        for i, m, n in zip(who, counts, keys):
            k, v = stored(held(i, n), dtype).astype(np.float64)
            for head in range(h):
                want, bound = ao.head(x[i][0][have[i]:n, head].astype(np.float64), k[:, head // 4], v[:, head // 4], ao.seen(m, n, True), d ** -0.5, dtype)["out"]
                assert (np.abs(got[first:first + m, head] - want) <= bound).all(), (i, head)
            first += m
            have[i] = n

    turn([37, 100, 1])
    turn([20, 0, 70])
    for step in range(3):
        new = [x[i][j][have[i]][None] for j in range(3) for i in range(3)]
        q, k, v = (np.concatenate(new[3 * j:3 * j + 3]) for j in range(3))
        c.write(k, v, np.array([slot(i, np.array([have[i]]))[0] for i in range(3)]))
        have = [n + 1 for n in have]
        dq, out = Array(device, q.shape, dtype, q), Array(device, q.shape, dtype)
        t, lengths = Ints(device, tables), Ints(device, have)
        decode.forward_device(caches[0], 3, dq.ptr, out.ptr, t.ptr, 10, lengths.ptr, longest=160)
        device.synchronize()
        got = out.get()
        for i in range(3):
            k, v = held(i, have[i])
            for head in range(h):
                want, bound = ao.head(q[i, head][None].astype(np.float64), k[:, head // 4], v[:, head // 4], np.ones((1, have[i]), bool), d ** -0.5,
                                      dtype, up=2.0 ** -16)["out"]
                assert (np.abs(got[i, head] - want[0]) <= bound[0]).all(), (step, i, head)
    for op in (prompt, decode, caches[0]):
        op.close()


# ---- captured, another stream, the same bits ----------------------------------------------------------------------------------------------------
class Step:
    """A prompt both ways, its keys to a cache and back, and new rows over it."""

    def __init__(self, device, seed=3):
        rng = np.random.default_rng(seed)
        self.device = device
        self.p = Problem(device, [200, 33, 129], 0, (8, 2, 64), "bf16", seed=seed)
        p = self.p
        A = lambda shape, t="bf16": Array(device, shape, t)  # noqa: E731
        self.out, self.lse = A(p.q.shape), A((8, p.rows), "f32")
        self.grads = [A(a.shape) for a in (p.q, p.k, p.v)]
        self.cache = rb.KvCache(device, 2, 64, 200, dtype="bf16", cache_dtype="int8")
        self.slots = Ints(device, rng.permutation(200 * 16)[:p.rows], np.int64)
        self.back = [A(p.k.shape) for _ in range(2)]
        self.decode = rb.DecodeAttention(device, 8, 2, 64, 3, dtype="bf16")
        self.tables, self.lengths = Ints(device, rng.permutation(200).reshape(2, 100)), Ints(device, [1600, 1203])
        self.new = A((2, 8, 64))

    def run(self):
        p = self.p
        p.op.forward_device(3, *p.inputs(), self.out.ptr, lse_ptr=self.lse.ptr, **p.where())
        p.op.backward_device(3, *p.inputs(), self.out.ptr, self.lse.ptr, p.dgo.ptr, *(g.ptr for g in self.grads), **p.where())
        self.cache.write_device(p.rows, p.dk.ptr, p.dv.ptr, self.slots.ptr)
        self.cache.read_device(p.rows, self.back[0].ptr, self.back[1].ptr, self.slots.ptr)
        self.decode.forward_device(self.cache, 2, p.dq.ptr, self.new.ptr, self.tables.ptr, 100, self.lengths.ptr, longest=1600)

    def results(self):
        self.device.synchronize()
        return [a.get() for a in (self.out, self.lse, *self.grads, *self.back, self.new)]


def same(a, b):
    return all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(a, b))


def test_a_captured_step_replays_like_the_eager_one(device, hip):  # noqa: F811
    eager, captured = Step(device), Step(device)
    cap = Capture(hip, device, captured.run)
    for turn in range(4):
        device.set_stream(None)
        lengths = np.array([1600 - 400 * turn, 1203 - 1 - 400 * turn], np.int32)  # (the graph was captured for the longest)
        for s in (eager, captured):
            s.lengths.buf.upload(np.concatenate([lengths, [0, 0]]).astype(np.int32))
        eager.run()
        want = eager.results()
        cap.replay()
        assert same(captured.results(), want)
        assert all(np.isfinite(a).all() for a in want)
    cap.close()


def test_on_a_stream_of_the_callers_own(device, hip):  # noqa: F811
    a, b = Step(device), Step(device)
    a.run()
    want = a.results()
    stream = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    try:
        device.set_stream(stream.value)
        b.run()
        got = b.results()
    finally:
        device.set_stream(None)
        hip.hipStreamDestroy(stream)
    assert same(got, want)


def test_the_same_call_gives_the_same_bits(device):
    s = Step(device)
    s.run()
    want = s.results()
    s.run()
    assert same(s.results(), want)


def test_operators_outlive_their_device_handle():
    dev = rb.Device.open(0)
    ops = [rb.Attention(dev, 4, 2, 64, backward_rows=10), rb.KvCache(dev, 2, 64, 4), rb.DecodeAttention(dev, 4, 2, 64, 2)]
    dev.close()
    for op in ops:
        op.close()


# ---- places that are not there, and not seen ------------------------------------------------------------------------------------------------------
def test_sequences_outside_the_arrays_are_cut(device):
    """Begins and counts below zero, behind the rows and near the largest number: what lies outside is cut off, nothing else is touched."""
    p = Problem(device, [40, 50, 30], 0, (4, 2, 64), "bf16")
    big = 2 ** 31 - 1
    begin, count = [0, 90, big, -5, 120, 40, 7], [40, big, 3, 0, 9, -7, -big]
    ints = [Ints(device, v) for v in (begin, count)]
    q, k, v, out, lse, go = p.q, p.k, p.v, Array(device, p.q.shape, "bf16"), Array(device, (4, p.rows), "f32"), p.dgo
    grads = [Array(device, a.shape, "bf16") for a in (q, k, v)]
    where = {**p.where(), "query_begin_ptr": ints[0].ptr, "query_count_ptr": ints[1].ptr}
    p.op.forward_device(len(begin), *p.inputs(), out.ptr, lse_ptr=lse.ptr, **where)
    p.op.backward_device(len(begin), *p.inputs(), out.ptr, lse.ptr, go.ptr, *(g.ptr for g in grads), **where)
    device.synchronize()
    want = p.wanted()
    for name in want:  # the sequence of rows 40 .. 90 is named by none
        value = want[name][0]
        (value[:, 40:90] if name == "lse" else value[40:90])[...] = np.nan
    check({"out": out.get(), "lse": lse.get(), **dict(zip(("grad_q", "grad_k", "grad_v"), (g.get() for g in grads)))}, want, "bf16")
    # launches for shorter sequences than there are: the first rows of each, as sequences of that length
    out = Array(device, p.q.shape, "bf16")
    p.op.forward_device(3, *p.inputs(), out.ptr, **{**p.where(), "longest_queries": 33, "longest_keys": 33})
    device.synchronize()
    got, first = out.get(), 0
    for n in (40, 50, 30):
        m = min(n, 33)
        for h in range(4):
            w, b = ao.head(*(a.astype(np.float64) for a in (q[first:first + m, h], k[first:first + m, h // 2], v[first:first + m, h // 2])), ao.seen(m, m, True),
                           p.scale, "bf16")["out"]
            assert (np.abs(got[first:first + m, h] - w) <= b).all()
        assert untouched(got[first + m:first + n], "bf16")
        first += n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,copies", [((4, 2, 64), 1), ((2, 2, 128), 1), ((16, 8, 64), 40)])
def test_what_a_row_does_not_see_has_no_effect(device, dtype, heads, copies):
    """Infinities and NaN in a key, in values and in a gradient: rows in front of them come out as without them, rows behind have them."""
    n, at = 150, 70
    p = Problem(device, [n] * copies, 0, heads, dtype)
    want = p.wanted()
    last = (copies - 1) * n  # the last sequence is spoilt
    v, go = p.v.copy(), p.go.copy()
    v[last + at, 0, 3], v[last + at + 1, 0, 5], v[last + at + 40, 0, 6] = np.nan, np.inf, -np.inf
    p.dv = Array(device, v.shape, dtype, v)
    out = p.forward()["out"]
    for col, row in ((3, at), (5, at + 1), (6, at + 40)):
        rows = out[last + row:, 0, col]
        # (f32 rows: an infinity may come out as NaN)
        assert np.isnan(rows).all() if col == 3 else (~np.isfinite(rows)).all() if dtype == "f32" else (rows == (np.inf if col == 5 else -np.inf)).all(), col
        out[last + row:, :heads[0] // heads[1], col] = np.nan
    hidden = np.isnan(out)
    keep = {"out": (np.where(hidden, 0, want["out"][0]), np.where(hidden, np.inf, want["out"][1]))}
    check({"out": np.where(hidden, 0, out)}, keep, dtype)
    # a key that is not seen: its scores are none; the rows that see it are NaN
    p.dv = Array(device, p.v.shape, dtype, p.v)
    k = p.k.copy()
    k[last + at, :, 1] = np.nan
    p.dk = Array(device, k.shape, dtype, k)
    got = p.forward()
    assert np.isnan(got["out"][last + at:]).all() and np.isnan(got["lse"][:, last + at:]).all()
    rows = np.arange(len(k)) < last + at
    check({"out": got["out"][rows], "lse": got["lse"][:, rows]},
          {"out": tuple(a[rows] for a in want["out"]), "lse": tuple(a[:, rows] for a in want["lse"])}, dtype)
    # backward: a gradient of NaN reaches its own row and the keys that this row sees
    p.dk = Array(device, p.k.shape, dtype, p.k)
    p.forward()
    go[last + at, :, 2] = np.nan
    p.dgo = Array(device, go.shape, dtype, go)
    got = p.backward()
    assert np.isnan(got["grad_q"][last + at]).all() and np.isnan(got["grad_k"][last:last + at + 1]).all()
    assert np.isnan(got["grad_v"][last:last + at + 1, :, 2]).all()
    clean = {"grad_q": np.arange(len(k)) != last + at, "grad_k": ~((np.arange(len(k)) >= last) & (np.arange(len(k)) <= last + at))}
    clean["grad_v"] = clean["grad_k"]
    check({n: got[n][clean[n]] for n in clean}, {n: tuple(a[clean[n]] for a in want[n]) for n in clean}, dtype)
    p.op.close()


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("bf16", "int8"), ("f32", "f32")])
@pytest.mark.parametrize("longest", [700, 3000])
def test_tables_and_lengths_that_name_places_outside(device, dtype, cache, longest):
    """Table entries that are no pages, lengths below zero, of zero and beyond the table, and slots outside the cache."""
    s = Sequences(device, [300, 100, 50, 64], (4, 2, 64), 16, dtype, cache, extra_pages=2)
    real, tables = s.lengths.copy(), s.tables.copy()
    s.lengths = np.array([300, 0, -5, 64], np.int32)
    s.check(s.run(longest=longest), lengths=[300, 0, 0, 64])
    assert (s.run(longest=longest)[1:3] == 0).all()
    s.tables[0, 3], s.tables[0, 7], s.tables[3, 0], s.lengths = -1, 2 ** 31 - 1, 10 ** 6, real
    s.check(s.run(longest=longest))
    s.tables[2, :] = -3
    assert (s.run(longest=longest)[2] == 0).all()
    s.tables, s.lengths = tables, np.array([2 ** 31 - 1, 100, 50, 64], np.int32)
    got = s.run(longest=longest)  # beyond the table, whose entries behind the sequence's pages are none: up to the end of its last page
    assert not np.array_equal(got[0], np.zeros_like(got[0]))
    got[0] = 0.0
    s.check(got, lengths=[0, 100, 50, 64])
    s.lengths = real
    s.check(s.run(longest=longest))
    s.lengths = np.minimum(real, 33).astype(np.int32)
    want = s.run()
    s.lengths = real
    got = s.run(longest=33)  # longer ones are cut
    assert np.array_equal(got, want)


@pytest.mark.parametrize("dtype,cache", [("bf16", "int8"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("count,longest", [(1500, 40), (1024, 1300), (1025, 1300), (300, 1100), (3, 9000)])
def test_many_sequences_and_long_ones(device, dtype, cache, count, longest):
    """A workgroup a sequence, and ranges over all of them; most are short, some have no row."""
    rng = np.random.default_rng(count)
    lengths = rng.integers(0, 41, count)
    lengths[rng.integers(0, count, 3)] = longest
    lengths[0], lengths[-1] = longest, longest - 1
    s = Sequences(device, lengths, (2, 1, 64), 16, dtype, cache)
    s.check(s.run())
    s.op.close()
    s.c.op.close()


# ---- offsets beyond 32 bits ------------------------------------------------------------------------------------------------------------------------
def test_rows_of_wide_strides_are_those_of_a_contiguous_call(device):
    """Rows 2^22 elements apart: 600 of them are 2^31 elements and more."""
    p = Problem(device, [500, 100], 0, (2, 1, 64), "bf16")
    want, grads = p.forward(), p.backward()
    stride, lib = 1 << 22, device._lib
    wide = [DeviceBuffer(device, 2 * ((p.rows - 1) * stride + a.shape[1] * 64)) for a in (p.q, p.k, p.v)]
    out = [DeviceBuffer(device, 2 * ((p.rows - 1) * stride + a.shape[1] * 64)) for a in (p.q, p.k, p.v)]

    def rows(buffers, copy):
        for b, a in zip(buffers, (p.q, p.k, p.v)):
            bits = synth.f32_to_bf16_bits(a).reshape(p.rows, -1)
            for r in range(p.rows):
                copy(b.ptr + 2 * r * stride, np.ascontiguousarray(bits[r]))

    def upload(at, row):
        assert lib.rbmoe_copy_to_device(device.handle, C.c_void_p(at), row.ctypes.data_as(C.c_void_p), row.nbytes) == 0

    try:
        rows(wide, upload)
        strides = dict(q_stride=stride, k_stride=stride, v_stride=stride)
        ptrs = [b.ptr for b in wide]
        o, l = Array(device, p.q.shape, "bf16"), Array(device, (2, p.rows), "f32")
        p.op.forward_device(2, *ptrs, o.ptr, lse_ptr=l.ptr, **{**p.where(), **strides})
        p.op.backward_device(2, *ptrs, o.ptr, l.ptr, p.dgo.ptr, *(b.ptr for b in out), **{**p.where(), **strides})
        device.synchronize()
        assert np.array_equal(o.get(), want["out"]) and np.array_equal(l.get(), want["lse"])
        for b, name in zip(out, ("grad_q", "grad_k", "grad_v")):
            for r in (0, 1, 499, 511, 512, p.rows - 1):
                row = np.empty(grads[name][r].size, np.uint16)
                assert lib.rbmoe_copy_to_host(device.handle, row.ctypes.data_as(C.c_void_p), C.c_void_p(b.ptr + 2 * r * stride), row.nbytes) == 0
                assert np.array_equal(synth.bf16_bits_to_f32(row), grads[name][r].reshape(-1)), (name, r)
    finally:
        for b in wide + out:
            b.free()


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "int8")])
def test_a_cache_of_more_than_four_gigabytes(device, dtype, cache):
    """Rows and sequences in its first, middle and last pages."""
    size = {"bf16": 2, "f32": 4, "int8": 1}[cache]
    kv, d, page = 4, 128, 16
    pages = (9 << 30) // (page * kv * d * 2 * size) + 3  # 9 GB: halves of pages on both sides of 2^32 and 2^33
    op = rb.KvCache(device, kv, d, pages, page_rows=page, dtype=dtype, cache_dtype=cache)
    rng = np.random.default_rng(1)
    table = np.array([[pages - 1, 0, pages // 2, pages - 2, pages // 3]], np.int32)
    n = 75
    at = np.arange(n)
    slots = table[0, at // page].astype(np.int64) * page + at % page
    k, v = rows_of(rng, n, kv, d, dtype), rows_of(rng, n, kv, d, dtype)
    small = Cache(device, kv, d, 5, page, dtype, cache)
    small.write(k, v, at)
    dk, dv, s = Array(device, k.shape, dtype, k), Array(device, v.shape, dtype, v), Ints(device, slots, np.int64)
    op.write_device(n, dk.ptr, dv.ptr, s.ptr)
    bk, bv = Array(device, k.shape, dtype), Array(device, v.shape, dtype)
    op.read_device(n, bk.ptr, bv.ptr, s.ptr)
    device.synchronize()
    assert np.array_equal(np.stack([bk.get(), bv.get()]), small.expected(at))
    q = Array(device, (1, 8, d), dtype, stored(rng.standard_normal((1, 8, d)), dtype))
    dec = rb.DecodeAttention(device, 8, kv, d, 1, dtype=dtype)
    got = []
    for c, t in ((op, table), (small.op, np.arange(5)[None])):
        out, tt, l = Array(device, (1, 8, d), dtype), Ints(device, t), Ints(device, [n])
        dec.forward_device(c, 1, q.ptr, out.ptr, tt.ptr, 5, l.ptr, longest=n)
        device.synchronize()
        got.append(out.get())
    assert np.array_equal(*got) and np.isfinite(got[0]).all()
    for o in (op, small.op, dec):
        o.close()


# ---- refusals ------------------------------------------------------------------------------------------------------------------------------------------
def test_refused_shapes(device):
    for heads, kv, d, dtype, error in ((8, 3, 64, "f32", rb.InvalidConfig), (0, 1, 64, "f32", rb.InvalidConfig), (4, 0, 64, "f32", rb.InvalidConfig),
                                       (4, 2, 0, "f32", rb.InvalidConfig), (4, 2, 60, "bf16", rb.Unsupported), (4, 2, 136, "bf16", rb.Unsupported),
                                       (2048, 2048, 64, "bf16", rb.Unsupported), (4, 2, 64, "int8", rb.InvalidConfig)):
        with pytest.raises(error):
            rb.Attention(device, heads, kv, d, dtype=dtype)
        with pytest.raises(error):
            rb.DecodeAttention(device, heads, kv, d, 4, dtype=dtype)
    with pytest.raises(rb.InvalidConfig):
        rb.Attention(device, 4, 2, 64, backward_rows=-1)
    with pytest.raises(rb.Unsupported):
        rb.Attention(device, 4, 2, 64, backward_rows=(1 << 30) + 1)
    for n, error in ((0, rb.InvalidConfig), (-1, rb.InvalidConfig), (65536, rb.Unsupported)):
        with pytest.raises(error):
            rb.DecodeAttention(device, 4, 2, 64, n)
    for page, pages, dtype, cache in ((8, 4, "f32", "f32"), (24, 4, "f32", "f32"), (8192, 4, "f32", "f32"), (16, 0, "f32", "f32"), (16, 4, "f32", "bf16"),
                                      (16, 4, "bf16", "f32"), (16, 4, "f32", "fp8")):
        with pytest.raises(rb.InvalidConfig):
            rb.KvCache(device, 2, 64, pages, page_rows=page, dtype=dtype, cache_dtype=cache)
    dev = rb.Device.open(0, budget_mib=1)
    try:
        with pytest.raises(rb.MemoryBudget):
            rb.KvCache(dev, 8, 128, 1000, dtype="f32")
        with pytest.raises(rb.MemoryBudget):
            rb.Attention(dev, 8, 8, 64, backward_rows=1 << 20)
        with pytest.raises(rb.MemoryBudget):
            rb.DecodeAttention(dev, 32, 8, 128, 1024)
    finally:
        dev.close()


def test_refused_calls(device):
    p = Problem(device, [20], 0, (4, 2, 64), "bf16")
    out, lse = Array(device, p.q.shape, "bf16"), Array(device, (4, 20), "f32")
    grads = [Array(device, a.shape, "bf16") for a in (p.q, p.k, p.v)]
    q, k, v = p.inputs()

    def forward(error, *at, n=1, **more):
        with pytest.raises(error):
            p.op.forward_device(n, *(at or (q, k, v, out.ptr)), **{**p.where(), **more})

    for i in range(4):
        at = [q, k, v, out.ptr]
        at[i] = 0
        forward(rb.InvalidInput, *at)
        at[i] = [q, k, v, out.ptr][i] + 1
        forward(rb.InvalidInput, *at)
    for more in (dict(q_stride=255), dict(k_stride=127), dict(v_stride=1), dict(scale=float("nan")), dict(scale=-1.0), dict(scale=float("inf")),
                 dict(query_rows=-1), dict(longest_keys=-1), dict(query_begin_ptr=0), dict(key_begin_ptr=p.ints[0].ptr),
                 dict(query_count_ptr=p.ints[1].ptr + 2), dict(lse_ptr=lse.ptr + 1)):
        forward(rb.InvalidInput, **more)
    forward(rb.InvalidInput, n=-1)
    forward(rb.Unsupported, n=65536)
    forward(rb.Unsupported, n=65535, query_rows=1 << 30, longest_queries=1 << 30)
    p.op.forward_device(0, 0, 0, 0, 0, **{**p.where(), "query_begin_ptr": 0, "query_count_ptr": 0})  # nothing to do
    p.op.forward_device(1, 0, 0, 0, 0, **{**p.where(), "longest_queries": 0})

    def backward(error, change=(), **more):
        at = [q, k, v, out.ptr, lse.ptr, p.dgo.ptr, *(g.ptr for g in grads)]
        for i, x in change:
            at[i] = x
        with pytest.raises(error):
            p.op.backward_device(1, *at, **{**p.where(), **more})

    for i in range(9):
        backward(rb.InvalidInput, [(i, 0)])
    for i in range(9):
        backward(rb.InvalidInput, [(i, [q, k, v, out.ptr, lse.ptr, p.dgo.ptr, *(g.ptr for g in grads)][i] + 1)])
    backward(rb.InvalidInput, [(7, grads[2].ptr)])
    backward(rb.InvalidInput, [(6, grads[2].ptr)])
    backward(rb.InvalidInput, query_rows=21)  # more than the workspace is for
    c = rb.KvCache(device, 2, 64, 4, dtype="bf16", cache_dtype="int8")
    slots = Ints(device, np.arange(4), np.int64)
    for call in (c.write_device, c.read_device):
        for args in ((-1, k, v, slots.ptr), (4, 0, v, slots.ptr), (4, k, 0, slots.ptr), (4, k, v, 0), (4, k + 1, v, slots.ptr), (4, k, v, slots.ptr + 4)):
            with pytest.raises(rb.InvalidInput):
                call(*args)
        with pytest.raises(rb.InvalidInput):
            call(4, k, v, slots.ptr, k_stride=100)
        with pytest.raises(rb.Unsupported):
            call((1 << 28) + 1, k, v, slots.ptr)
        call(0, 0, 0, 0)
    with pytest.raises(rb.InvalidInput):
        c.read_device(4, grads[1].ptr, grads[1].ptr, slots.ptr)
    d = rb.DecodeAttention(device, 4, 2, 64, 2, dtype="bf16")
    t, l = Ints(device, np.zeros((2, 4))), Ints(device, [1, 1])
    for cache, args, more in ((c, (3, q, out.ptr, t.ptr, 4, l.ptr), {}), (c, (-1, q, out.ptr, t.ptr, 4, l.ptr), {}), (c, (2, 0, out.ptr, t.ptr, 4, l.ptr), {}),
                              (c, (2, q, 0, t.ptr, 4, l.ptr), {}), (c, (2, q, out.ptr, 0, 4, l.ptr), {}), (c, (2, q, out.ptr, t.ptr, 4, 0), {}),
                              (c, (2, q + 1, out.ptr, t.ptr, 4, l.ptr), {}), (c, (2, q, out.ptr, t.ptr + 1, 4, l.ptr), {}),
                              (c, (2, q, out.ptr, t.ptr, -1, l.ptr), {}), (c, (2, q, out.ptr, t.ptr, 4, l.ptr), dict(longest=-1)),
                              (c, (2, q, out.ptr, t.ptr, 4, l.ptr), dict(q_stride=255)), (c, (2, q, out.ptr, t.ptr, 4, l.ptr), dict(scale=-0.5)),
                              (rb.KvCache(device, 1, 64, 4, dtype="bf16"), (2, q, out.ptr, t.ptr, 4, l.ptr), {}),
                              (rb.KvCache(device, 2, 32, 4, dtype="bf16"), (2, q, out.ptr, t.ptr, 4, l.ptr), {}),
                              (rb.KvCache(device, 2, 64, 4, dtype="f32"), (2, q, out.ptr, t.ptr, 4, l.ptr), {})):
        with pytest.raises(rb.InvalidInput):
            d.forward_device(cache, *args, **{"longest": 4, **more})
    d.forward_device(c, 2, q, out.ptr, 0, 0, l.ptr, longest=4)  # no pages at all: zeros
    device.synchronize()
    assert (out.get()[:2] == 0).all() and untouched(out.get()[2:], "bf16")
    other = rb.Device.open(0)
    with pytest.raises(rb.InvalidInput):
        d.forward_device(rb.KvCache(other, 2, 64, 4, dtype="bf16"), 2, q, out.ptr, t.ptr, 4, l.ptr, longest=4)
    other.close()
