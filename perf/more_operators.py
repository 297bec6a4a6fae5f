"""Timed operators of a block's attention: what stands beside the mixture-of-experts layer in a training or serving step.

* ``prompt`` / ``prompt_backward`` — attention of whole sequences, packed one behind the other, with grouped heads (``Attention``);
* ``cache`` — rows of keys and values written to a paged cache, as they are or in 8 bits, and read back (``KvCache``);
* ``decode`` — a serving step: every sequence's new row is written to the cache, then attends to all of its sequence (``DecodeAttention``).

Heads are those of the default ``TransformerConfig`` (8 heads in groups of 4, 64 elements each) and the common layouts of larger models (16 and
32 heads in groups of 4, 128 elements); drawn ones also have other groups and widths.  Sequences have 1 to 16384 rows, caches up to 131072.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4, "int8": 1}


def _prompt(kind, sequences, longest, heads, dtype, earlier=0, causal=True, fused=True, **more):
    """`longest`: rows of the longest sequence, the others are shorter; `earlier`: keys that stand in front of the longest one's rows."""
    h, kv, d = heads
    return dict(kind=kind, sequences=sequences, longest=longest, heads=h, kv_heads=kv, head_dim=d, dtype=dtype, earlier=earlier,
                causal=causal, fused=fused, **more)


def _cached(kind, sequences, longest, heads, dtype, cache, page=16, padding=0.0, **more):
    h, kv, d = heads
    return dict(kind=kind, sequences=sequences, longest=longest, heads=h, kv_heads=kv, head_dim=d, dtype=dtype, cache=cache, page=page,
                padding=padding, **more)


_DEFAULT, _MIDDLE, _LARGE = (8, 2, 64), (16, 4, 128), (32, 8, 128)


def listed():
    return [
        # one short prompt of the default model: all latency
        _prompt("prompt", 1, 77, _DEFAULT, "bf16", name="prompt_short"),
        # a training micro-batch in the reference's own precision, sequences of every length up to the default model's
        _prompt("prompt", 6, 2048, _DEFAULT, "f32", name="prompt_f32_packed"),
        # new rows of conversations whose first turns are in the cache already (read back as rows: not fused with the queries)
        _prompt("prompt", 5, 513, _LARGE, "bf16", earlier=4000, fused=False, name="prompt_continued"),
        # one long prompt
        _prompt("prompt", 1, 16384, _MIDDLE, "bf16", name="prompt_long"),
        # a training micro-batch of the default model, ragged
        _prompt("prompt_backward", 8, 2048, _DEFAULT, "bf16", name="prompt_backward_packed"),
        # a few sequences in the reference's own precision
        _prompt("prompt_backward", 3, 700, _DEFAULT, "f32", name="prompt_backward_f32"),
        # one long sequence of a larger model
        _prompt("prompt_backward", 1, 8192, _MIDDLE, "bf16", name="prompt_backward_long"),
        # the rows of a serving step of short prompts and new tokens, padded to the batch
        _cached("cache", 9, 100, _DEFAULT, "bf16", "bf16", padding=0.1, name="cache_step"),
        # prompts into a cache of 8 bits
        _cached("cache", 12, 4096, _LARGE, "bf16", "int8", page=64, name="cache_prompts_int8"),
        # one conversation with the default model: all latency
        _cached("decode", 1, 777, _DEFAULT, "bf16", "bf16", name="decode_one"),
        # a serving batch of conversations of all lengths over a cache of 8 bits
        _cached("decode", 64, 8192, _LARGE, "bf16", "int8", name="decode_batch_int8"),
        # a few very long ones
        _cached("decode", 4, 131072, _LARGE, "bf16", "bf16", page=64, name="decode_long"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        h, kv, d = rng.choice([_DEFAULT, _DEFAULT, _MIDDLE, _LARGE, (8, 8, 64), (6, 3, 80), (12, 1, 96), (5, 5, 40), (32, 4, 64), (24, 2, 128)])
        kind = rng.choice(["prompt", "prompt", "prompt_backward", "prompt_backward", "cache", "decode", "decode"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        n = _log_int(rng, 1, 64)
        if kind.startswith("prompt"):
            longest = _log_int(rng, 1, 8192)
            c = _prompt(kind, min(n, 24), longest, (h, kv, d), dtype, earlier=rng.choice([0, 0, _log_int(rng, 1, 4096)]),
                        causal=rng.random() < 0.8, fused=rng.random() < 0.5)
            # (of the plain form, which keeps every score)
            scores = c["sequences"] * h * longest * (longest + c["earlier"])
            if scores <= (1 << 30) and work(c)["flops"] <= (2e11 if dtype == "f32" else 1.5e12):
                return c
            continue
        c = _cached(kind, n, _log_int(rng, 1, 4096 if kind == "cache" else 32768), (h, kv, d), dtype, rng.choice([dtype, "int8"]),
                    page=rng.choice([16, 32, 64, 128]), padding=rng.choice([0.0, 0.1]) if kind == "cache" else 0.0)
        if sum(_lengths(c)) * kv * d <= (3.5e7 if kind == "cache" else 2.5e8):
            return c


def _lengths(c):
    """Rows of each sequence: the first is the longest, the others anything from one row on."""
    rng = random.Random("%d of %d" % (c["sequences"], c["longest"]))
    return [c["longest"]] + [rng.randint(1, c["longest"]) for _ in range(c["sequences"] - 1)]


def _earlier(c):
    """Keys in front of each sequence's rows."""
    rng = random.Random("%d behind %d" % (c["sequences"], c["earlier"]))
    return [c["earlier"]] + [rng.randint(0, c["earlier"]) for _ in range(c["sequences"] - 1)]


# ----------------------------------------------------------------------------- inputs
def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, device="cuda", dtype=dtype)


def _starts(counts):
    at, got = 0, []
    for n in counts:
        got.append(at)
        at += n
    return got


class _State:
    pass


def _keys(g, rows, kv, d):
    """Keys share a direction within a head, and some channels are larger than others."""
    return (_normal(g, (rows, kv, d)) + _normal(g, (1, kv, d))) * torch.exp(_normal(g, (1, kv, d), 0.4))


def _values(g, rows, kv, d):
    return _normal(g, (rows, kv, d)) + _normal(g, (1, kv, d), 0.5)


def _inputs(case, seed):
    """The tensors that a user's program has in hand before the call."""
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = _State()
    s.case = c
    t, h, kv, d = _TORCH[c["dtype"]], c["heads"], c["kv_heads"], c["head_dim"]
    s.scale = 1.0 / math.sqrt(d)
    order = random.Random(int(seed))
    counts = _lengths(c)
    if c["kind"].startswith("prompt"):
        both = list(zip(counts, _earlier(c)))
        order.shuffle(both)
        counts, keys = [n for n, _ in both], [n + e for n, e in both]
        s.rows, s.key_rows = sum(counts), sum(keys)
        s.counts, s.key_counts = counts, keys
        s.begin, s.count, s.key_begin, s.key_count = map(_ints, (_starts(counts), counts, _starts(keys), keys))
        q, k, v = _normal(g, (s.rows, h, d), 1.2), _keys(g, s.key_rows, kv, d), _values(g, s.key_rows, kv, d)
        if c["fused"] and not c["earlier"]:  # as one projection leaves them
            s.fused = torch.cat([q, k, v], dim=1).to(t)
            s.q, s.k, s.v = s.fused[:, :h], s.fused[:, h:h + kv], s.fused[:, h + kv:]
        else:
            s.q, s.k, s.v = q.to(t), k.to(t), v.to(t)
        if c["kind"] == "prompt_backward":
            s.out, s.lse = _prompt_plain(s)
            s.out = s.out.to(t)
            s.grad_out = _normal(g, (s.rows, h, d), 1e-2).to(t)
        return s
    order.shuffle(counts)
    page = c["page"]
    pages = [-(-n // page) for n in counts]
    s.pages = sum(pages) + 3  # a few pages of the pool are free
    s.table_pages = max(pages)
    places = torch.randperm(s.pages, generator=g, device="cuda")
    first = _ints(_starts(pages), torch.int64)
    s.counts, s.lengths, s.rows = counts, _ints(counts), sum(counts)
    column = torch.arange(s.table_pages, device="cuda")[None]
    s.tables = torch.where(column < _ints(pages, torch.int64)[:, None], places[(first[:, None] + column).clamp(max=s.pages - 1)], 0).to(torch.int32)
    sequence = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), _ints(counts, torch.int64))
    at = torch.arange(s.rows, device="cuda") - _ints(_starts(counts), torch.int64)[sequence]
    s.slots = s.tables[sequence, at // page].long() * page + at % page
    s.k, s.v = _keys(g, s.rows, kv, d).to(t), _values(g, s.rows, kv, d).to(t)
    if c["kind"] == "cache":
        n = round(c["padding"] * s.rows)
        if n:
            s.slots[torch.randperm(s.rows, generator=g, device="cuda")[:n]] = -1
        return s
    s.q = _normal(g, (len(counts), h, d), 1.2).to(t)
    s.new_k, s.new_v = _keys(g, len(counts), kv, d).to(t), _values(g, len(counts), kv, d).to(t)
    last = s.lengths.long() - 1
    s.new_slots = s.tables.gather(1, (last // page)[:, None])[:, 0].long() * page + last % page
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = case
    if own:
        import rustingbrain_amd as rb
        device = _device(rb)
        if c["kind"].startswith("prompt"):
            s.handle = rb.Attention(device, c["heads"], c["kv_heads"], c["head_dim"], dtype=c["dtype"],
                                    backward_rows=s.rows if c["kind"] == "prompt_backward" else 0)
            if c["kind"] == "prompt":
                s.out = torch.empty(s.rows, c["heads"], c["head_dim"], dtype=s.q.dtype, device="cuda")
                s.lse = torch.empty(c["heads"], s.rows, device="cuda")
            elif c["fused"] and not c["earlier"]:  # gradients lie as their inputs do
                s.grad = torch.empty_like(s.fused)
                h, kv = c["heads"], c["kv_heads"]
                s.grad_q, s.grad_k, s.grad_v = s.grad[:, :h], s.grad[:, h:h + kv], s.grad[:, h + kv:]
            else:
                s.grad_q, s.grad_k, s.grad_v = torch.empty_like(s.q), torch.empty_like(s.k), torch.empty_like(s.v)
        else:
            s.cache = rb.KvCache(device, c["kv_heads"], c["head_dim"], s.pages, page_rows=c["page"], dtype=c["dtype"], cache_dtype=c["cache"])
            if c["kind"] == "cache":
                s.got_k, s.got_v = torch.empty_like(s.k), torch.empty_like(s.v)
            else:
                torch.cuda.synchronize()
                s.cache.write_device(s.rows, s.k.data_ptr(), s.v.data_ptr(), s.slots.data_ptr())
                s.handle = rb.DecodeAttention(device, c["heads"], c["kv_heads"], c["head_dim"], len(s.counts), dtype=c["dtype"])
                s.out = torch.empty_like(s.q)
                device.synchronize()
    elif not c["kind"].startswith("prompt"):
        s.pool = _pool(s)
        if c["kind"] == "decode":
            _write(s, s.k, s.v, s.slots)
    if c["kind"] == "decode":
        s.k = s.v = None  # they are in the cache
    torch.cuda.synchronize()
    return s


_handle = None


def _device(rb):
    """One handle for the GPU, as a program with many layers keeps."""
    global _handle
    if _handle is None:
        _handle = rb.Device.open(0)
    return _handle


# ----------------------------------------------------------------------------- one pass, plain
def _padded(t, begin, count, longest):
    """[sequences, longest, heads, d] in 32 bits, zeros behind each sequence, and which of its rows are there."""
    at = torch.arange(longest, device=t.device)[None]
    live = at < count[:, None]
    rows = torch.where(live, begin[:, None] + at, 0).long()
    return torch.where(live[:, :, None, None], t[rows].float(), 0.0), live


def _row_places(begin, rows, longest):
    """Where each packed row lies in the padded layout."""
    row = torch.arange(rows, device=begin.device, dtype=torch.int32)
    sequence = torch.searchsorted(begin.contiguous(), row, right=True) - 1
    return sequence * longest + row - begin[sequence]


def _by_group(t, kv):
    """[n, longest, heads, d] -> [n kv, group longest, d]"""
    n, length, h, d = t.shape
    return t.view(n, length, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n * kv, h // kv * length, d)


def _from_group(t, n, kv, length):
    """[n kv, group longest, d] -> [n longest, heads, d]"""
    d = t.shape[-1]
    return t.view(n, kv, -1, length, d).permute(0, 3, 1, 2, 4).reshape(n * length, -1, d)


def _prompt_scores(s):
    c = s.case
    kv, lq, lk = c["kv_heads"], max(s.counts), max(s.key_counts)
    q, _ = _padded(s.q, s.begin, s.count, lq)
    k, live = _padded(s.k, s.key_begin, s.key_count, lk)
    v, _ = _padded(s.v, s.key_begin, s.key_count, lk)
    q, k, v = _by_group(q, kv), _by_group(k, kv), _by_group(v, kv)
    n, group = len(s.counts), c["heads"] // kv
    scores = (torch.matmul(q, k.mT.contiguous()) * s.scale).view(n, kv, group, lq, lk)
    seen = live[:, None, :]
    if c["causal"]:
        i, j = torch.arange(lq, device=q.device)[:, None], torch.arange(lk, device=q.device)[None]
        seen = seen & (j <= i + (s.key_count - s.count)[:, None, None])
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    return q, k, v, scores


def _prompt_plain(s):
    c = s.case
    n, kv, lq = len(s.counts), c["kv_heads"], max(s.counts)
    _, _, v, scores = _prompt_scores(s)
    most = scores.amax(dim=-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    p = torch.exp(scores - most)
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p.view(n * kv, -1, v.shape[1]), v) / torch.where(total == 0, 1.0, total).view(n * kv, -1, 1)
    lse = (torch.log(total) + most).view(n * kv, -1, 1)
    place = _row_places(s.begin, s.rows, lq)
    return _from_group(out, n, kv, lq)[place], _from_group(lse, n, kv, lq)[place][:, :, 0].mT.contiguous()


def _prompt_backward_plain(s):
    c = s.case
    n, kv, lq, lk = len(s.counts), c["kv_heads"], max(s.counts), max(s.key_counts)
    q, k, v, scores = _prompt_scores(s)
    do, _ = _padded(s.grad_out, s.begin, s.count, lq)
    lse, live = _padded(s.lse.mT[:, :, None], s.begin, s.count, lq)
    do, lse = _by_group(do, kv), _by_group(lse, kv)
    p = torch.exp(scores.view(n * kv, -1, lk) - lse)
    p = torch.where(live[:, None, None, :].expand(n, kv, c["heads"] // kv, lq).reshape(n * kv, -1, 1), p, 0.0)
    dp = torch.matmul(do, v.mT.contiguous())
    ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) * s.scale
    grad_v, grad_k = torch.matmul(p.mT.contiguous(), do), torch.matmul(ds.mT.contiguous(), q)
    place, key_place = _row_places(s.begin, s.rows, lq), _row_places(s.key_begin, s.key_rows, lk)
    t = s.q.dtype
    return {"grad_q": _from_group(torch.matmul(ds, k), n, kv, lq)[place].to(t), "grad_k": _from_group(grad_k, n, kv, lk)[key_place].to(t),
            "grad_v": _from_group(grad_v, n, kv, lk)[key_place].to(t)}


def _pool(s):
    c = s.case
    rows, kv, d = s.pages * c["page"] + 1, c["kv_heads"], c["head_dim"]  # (one more for rows without a place)
    store = torch.int8 if c["cache"] == "int8" else _TORCH[c["cache"]]
    p = {name: torch.zeros(rows, kv, d, dtype=store, device="cuda") for name in "kv"}
    if c["cache"] == "int8":
        p.update({name + "_scale": torch.zeros(rows, kv, 1, device="cuda") for name in "kv"})
    return p


def _write(s, k, v, slots):
    slots = torch.where(slots < 0, s.pages * s.case["page"], slots)
    k, v = k.float(), v.float()
    if s.case["cache"] == "int8":
        k_most, v_most = k.abs().amax(dim=2, keepdim=True), v.abs().amax(dim=2, keepdim=True)
        s.pool["k_scale"][slots], s.pool["v_scale"][slots] = k_most / 127.0, v_most / 127.0
        k, v = torch.round(k * 127.0 / k_most), torch.round(v * 127.0 / v_most)
    s.pool["k"][slots], s.pool["v"][slots] = k.to(s.pool["k"].dtype), v.to(s.pool["v"].dtype)


def _stored(s, name, slots):
    got = s.pool[name][slots].float()
    return got * s.pool[name + "_scale"][slots] if s.case["cache"] == "int8" else got


def _decode_plain(s):
    c = s.case
    n, kv, h, page = len(s.counts), c["kv_heads"], c["heads"], c["page"]
    _write(s, s.new_k, s.new_v, s.new_slots)
    slots = (s.tables.long()[:, :, None] * page + torch.arange(page, device=s.q.device)).view(n, -1)
    k, v = _stored(s, "k", slots), _stored(s, "v", slots)
    live = (torch.arange(slots.shape[1], device=s.q.device)[None] < s.lengths[:, None])[:, None, None]
    k, v = k.permute(0, 2, 3, 1).contiguous(), torch.where(live.view(n, -1, 1, 1), v, 0.0).permute(0, 2, 1, 3).contiguous()
    scores = torch.where(live, torch.matmul(s.q.float().view(n, kv, h // kv, -1), k) * s.scale, -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)).view(n, h, -1).to(s.q.dtype)


def run(state):
    s, c = state, state.case
    kind = c["kind"]
    if own:
        if kind.startswith("prompt"):
            where = dict(query_begin_ptr=s.begin.data_ptr(), query_count_ptr=s.count.data_ptr(), key_begin_ptr=s.key_begin.data_ptr(),
                         key_count_ptr=s.key_count.data_ptr(), query_rows=s.rows, key_rows=s.key_rows, longest_queries=max(s.counts),
                         longest_keys=max(s.key_counts), q_stride=s.q.stride(0), k_stride=s.k.stride(0), v_stride=s.v.stride(0),
                         causal=c["causal"], scale=s.scale)
            if kind == "prompt":
                s.handle.forward_device(len(s.counts), s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.out.data_ptr(),
                                        lse_ptr=s.lse.data_ptr(), **where)
                return {"out": s.out, "lse": s.lse}
            s.handle.backward_device(len(s.counts), s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.out.data_ptr(), s.lse.data_ptr(),
                                     s.grad_out.data_ptr(), s.grad_q.data_ptr(), s.grad_k.data_ptr(), s.grad_v.data_ptr(), **where)
            return {"grad_q": s.grad_q, "grad_k": s.grad_k, "grad_v": s.grad_v}
        if kind == "cache":
            s.cache.write_device(s.rows, s.k.data_ptr(), s.v.data_ptr(), s.slots.data_ptr())
            s.cache.read_device(s.rows, s.got_k.data_ptr(), s.got_v.data_ptr(), s.slots.data_ptr())
            return {"k": s.got_k, "v": s.got_v}
        s.cache.write_device(len(s.counts), s.new_k.data_ptr(), s.new_v.data_ptr(), s.new_slots.data_ptr())
        s.handle.forward_device(s.cache, len(s.counts), s.q.data_ptr(), s.out.data_ptr(), s.tables.data_ptr(), s.table_pages,
                                s.lengths.data_ptr(), longest=max(s.counts), scale=s.scale)
        return s.out
    if kind == "prompt":
        out, lse = _prompt_plain(s)
        return {"out": out.to(s.q.dtype), "lse": lse}
    if kind == "prompt_backward":
        return _prompt_backward_plain(s)
    if kind == "cache":
        _write(s, s.k, s.v, s.slots)
        there = (s.slots >= 0)[:, None, None]
        slots = s.slots.clamp(min=0)
        return {"k": torch.where(there, _stored(s, "k", slots), 0.0).to(s.k.dtype),
                "v": torch.where(there, _stored(s, "v", slots), 0.0).to(s.v.dtype)}
    return _decode_plain(s)


# ----------------------------------------------------------------------------- in 64 bits
def _exact_prompt(s):
    """Sequence by sequence and head by head; gradients by differentiating the forward."""
    c = s.case
    group = c["heads"] // c["kv_heads"]
    backward = c["kind"] == "prompt_backward"
    if backward:
        got = {"grad_q": torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")}
        got.update({n: torch.zeros(s.k.shape, dtype=torch.float64, device="cuda") for n in ("grad_k", "grad_v")})
    else:
        got = {"out": torch.zeros(s.q.shape, dtype=torch.float64, device="cuda"),
               "lse": torch.zeros(c["heads"], s.rows, dtype=torch.float64, device="cuda")}
    for a, n, b, m in zip(_starts(s.counts), s.counts, _starts(s.key_counts), s.key_counts):
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1) if c["causal"] else None
        for h in range(c["heads"]):
            q, k, v = (t.double().contiguous().requires_grad_(backward)
                       for t in (s.q[a:a + n, h], s.k[b:b + m, h // group], s.v[b:b + m, h // group]))
            with torch.set_grad_enabled(backward):
                x = s.scale * torch.mm(q, k.t())
                x = x if hidden is None else x.masked_fill(hidden, -math.inf)
                out = torch.mm(torch.softmax(x, dim=1), v)
            if backward:
                for name, grad, at, head in zip(got, torch.autograd.grad(out, (q, k, v), s.grad_out[a:a + n, h].double()), (a, b, b),
                                                (h, h // group, h // group)):
                    got[name][at:at + grad.shape[0], head] += grad
            else:
                got["out"][a:a + n, h], got["lse"][h, a:a + n] = out, torch.logsumexp(x, dim=1)
    return got


def _exact_stored(t, cache):
    """The values that a cache holds for rows [.., d]."""
    t = t.double()
    if cache != "int8":
        return t
    most = torch.linalg.vector_norm(t, ord=math.inf, dim=-1, keepdim=True)
    return torch.round(127.0 * t / most) * (most / 127.0)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"].startswith("prompt"):
        return _exact_prompt(s)
    if case["kind"] == "cache":
        there = (s.slots >= 0).double()[:, None, None]
        return {"k": _exact_stored(s.k, case["cache"]) * there, "v": _exact_stored(s.v, case["cache"]) * there}
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for i, (a, n) in enumerate(zip(_starts(s.counts), s.counts)):
        for h in range(case["kv_heads"]):
            k, v = (_exact_stored(torch.cat([old[a:a + n - 1, h], new[i:i + 1, h]]), case["cache"])
                    for old, new in ((s.k, s.new_k), (s.v, s.new_v)))
            heads = slice(h * group, (h + 1) * group)
            out[i, heads] = torch.mm(torch.softmax(s.scale * torch.mm(s.q[i, heads].double(), k.t()), dim=1), v)
    return out


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    h, kv, d, size = c["heads"], c["kv_heads"], c["head_dim"], _SIZE[c["dtype"]]
    counts = _lengths(c)
    rows = float(sum(counts))
    if c["kind"].startswith("prompt"):
        earlier = _earlier(c)
        key_rows = rows + sum(earlier)
        pairs = float(sum(n * e + (n * (n + 1) // 2 if c["causal"] else n * n) for n, e in zip(counts, earlier)))
        if c["kind"] == "prompt":
            return {"bytes": (2.0 * h * rows + 2.0 * kv * key_rows) * d * size + 4.0 * h * rows, "flops": 4.0 * d * h * pairs}
        return {"bytes": (4.0 * h * rows + 4.0 * kv * key_rows) * d * size + 4.0 * h * rows, "flops": 10.0 * d * h * pairs}
    row = 2.0 * kv * d * _SIZE[c["cache"]] + (8.0 * kv if c["cache"] == "int8" else 0.0)  # of the cache
    if c["kind"] == "cache":
        return {"bytes": 2.0 * rows * (2.0 * kv * d * size + row + 8.0), "flops": 8.0 * rows * kv * d}
    n = float(c["sequences"])
    return {"bytes": rows * row + n * (row + 2.0 * kv * d * size + 2.0 * h * d * size), "flops": 4.0 * d * h * rows}
