"""How exact attention is in a given arithmetic: the formulas with a choice of matrix product and of what is rounded on the way, and errors in the
Frobenius norm beside 64 bits.

f32 rows.  The kernels multiply in parts that keep 24 bits, leave out products below 2^-25 of a term, and otherwise round where the formula in f32
rounds: sums of products, the exponential's argument, the exponential, the quotient.  Such errors are of the size of f32's own and
independent of them, so a result may be sqrt(2) times as far from 64 bits as the formula in f32 (numpy) is on the same input, 1.5 with
the chance of a finite sample.  What is exact in f32 by chance (a row of one key) may be off by a rounding, 2^-24 of the result's norm.

bf16 rows.  p and ds are rounded to bf16 for their products, results once more; everything else is f32, a thousand times finer, and the error that stored
rows leave in delta is mended.  So errors are those of these roundings on the exact p and ds (`bf16_rounded`).  They are independent, some hundred of
them at least: the norms of two such sets differ by a few percent by chance, 1.2 is allowed."""
import numpy as np

from rustingbrain_amd import synth

NAMES = ("out", "lse", "grad_q", "grad_k", "grad_v")


def formulas(q, k, v, go, mask, scale, product=np.matmul):
    """{name: array} in the type of the arguments."""
    kind = q.dtype.type
    s = np.where(mask, kind(scale) * product(q, k.T), kind(-np.inf))
    top = s.max(axis=1, keepdims=True)
    e = np.exp(s - top)
    total = e.sum(axis=1, keepdims=True)
    out, lse = product(e, v) / total, np.log(total) + top
    p = np.exp(s - lse)
    ds = p * (product(go, v.T) - (go * out).sum(axis=1, keepdims=True))
    grads = kind(scale) * product(ds, k), kind(scale) * product(ds.T, q), product(p.T, go)
    got = dict(zip(NAMES, (out, lse[:, 0], *grads)))
    assert all(a.dtype == kind for a in got.values())
    return got


def rounded(x):
    return synth.round_bf16(np.asarray(x, np.float32)).astype(np.float64)


def bf16_rounded(q, k, v, go, mask, scale, mended=True):
    """The results in 64 bits with p and ds as bf16 operands, before their own rounding.  A row's ds add up to zero, and what rounding adds to that
    sum is taken off again in proportion to p; `mended` False: as if neither that nor delta, from rows as they are stored, were mended."""
    f = formulas(q, k, v, go, mask, scale)
    s = np.where(mask, scale * (q @ k.T), -np.inf)
    e, p = np.exp(s - s.max(axis=1, keepdims=True)), np.exp(s - f["lse"][:, None])
    out = rounded(e) @ v / e.sum(axis=1, keepdims=True)
    delta = (go * (f["out"] if mended else rounded(out))).sum(axis=1, keepdims=True)
    ds = rounded(p * (go @ v.T - delta))
    ds[mask.sum(axis=1) == 1] = 0.0
    grad_q = ds @ k - (ds.sum(axis=1, keepdims=True) * (p @ k) if mended else 0.0)
    return dict(zip(NAMES, (out, f["lse"], scale * grad_q, scale * ds.T @ q, rounded(p).T @ go)))


def in_parts(parts, dropped):
    """A product of operands in so many bf16 parts (64-bit arrays), of which those beside each other by `dropped` or more are left out."""
    def cut(x):
        got = []
        for _ in range(parts):
            got.append(synth.round_bf16(x.astype(np.float32)).astype(np.float64))
            x = x - got[-1]
        return got

    def product(a, b):
        a, b = cut(a), cut(b)
        return sum(a[i] @ b[j] for i in range(parts) for j in range(parts) if i + j < dropped)
    return product


def rows(rng, nq, nk, d):
    """q, k, v, grad_out in f32; keys and values share a direction."""
    x = lambda n: rng.standard_normal((n, d))  # noqa: E731
    return [a.astype(np.float32) for a in (1.3 * x(nq), x(nk) + 1.5 * x(1), x(nk) + 0.5 * x(1), 0.1 * x(nq))]


def error(got, want):
    return np.linalg.norm(np.asarray(got, np.float64) - want), np.linalg.norm(want)


def as_exact_as_f32(got, f32, want, factor=1.5, least=2.0 ** -24):
    """Names of results that are further from 64 bits than the formula in f32 allows, with their errors."""
    bad = {}
    for name in got:
        (err, norm), (own, _) = error(got[name], want[name]), error(f32[name], want[name])
        if not err <= max(factor * own, least * norm):
            bad[name] = (err / norm, own / norm)
    return bad


def as_exact_as_bf16(got, model, want):
    """The same for results of bf16 rows (`model`: bf16_rounded, rounded once more); lse is f32 and held elsewhere."""
    names = [n for n in got if n != "lse"]
    return as_exact_as_f32({n: got[n] for n in names}, {n: rounded(model[n]) for n in names}, want, 1.2, 2.0 ** -9)
