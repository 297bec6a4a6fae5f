"""Attention of whole sequences in 64 bits, and how far a result of f32 sums over operands of `dtype` may be off it.

Bounds.  u is half a step of the type (2^-8 bf16, 2^-24 f32), up what p and ds lose as operands of the second product (2^-8 bf16, nothing f32).
A score is a sum of d products: off by (d + 8) 2^-24 of the sum of their magnitudes, and 2^-21 of itself in the exponent's argument (its
factor, its product and difference each a rounding, the exponential two steps); e is a row's largest.  p is off by twice that (its own score's, and
those in the row's sum), a sum of n terms by (n + 40) 2^-24 of their magnitudes."""
import numpy as np

F = 2.0 ** -24


def seen(nq, nk, causal):
    i, j = np.arange(nq)[:, None], np.arange(nk)[None]
    return (j <= i + nk - nq) if causal else np.ones((nq, nk), bool)


def softmax(s, mask):
    """p and lse of the rows of s over the places of mask; what lies elsewhere in s is not used."""
    s = np.where(mask, s, -np.inf)
    top = s.max(axis=1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = p.sum(axis=1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = np.log(total)[:, 0] + np.where(np.isfinite(top), top, 0.0)[:, 0]
    return p / np.where(total == 0, 1.0, total), lse


def head(q, k, v, mask, scale, dtype, grad_out=None, up=None):
    """{name: (value, bound)} of one head of one sequence, all inputs [rows, d] in 64 bits."""
    u, base = (2.0 ** -8, 2.0 ** -8) if dtype == "bf16" else (F, 0.0)
    up = base if up is None else up
    d, nk = q.shape[1], k.shape[0]
    s = scale * (q @ k.T)
    p, lse = softmax(s, mask)
    e_s = np.where(mask, (d + 8) * F * scale * (np.abs(q) @ np.abs(k).T) + 2.0 ** -21 * np.abs(s), 0.0)
    e = 2 * e_s.max(axis=1, keepdims=True, initial=0.0) + (nk + 40) * F
    out = p @ v
    off = u * np.abs(out) + (up + e) * (p @ np.abs(v))
    got = {"out": (out, 1.01 * off + 1e-37), "lse": (lse, 1.01 * (e[:, 0] + 2.0 ** -21 * (np.abs(np.where(np.isfinite(lse), lse, 0)) + 1)))}
    if grad_out is None:
        return got
    rows = q.shape[0]
    e = e + 2.0 ** -21 * (np.abs(np.where(np.isfinite(lse), lse, 0.0))[:, None] + 1)  # (lse was rounded)
    dp, ao = grad_out @ v.T, np.abs(grad_out)
    delta = (p * dp).sum(axis=1, keepdims=True)
    ds = p * (dp - delta)
    e_dp = (d + 8) * F * (ao @ np.abs(v).T)
    e_out = (ao * off).sum(axis=1, keepdims=True) + (d + 8) * F * (ao * np.abs(out)).sum(axis=1, keepdims=True)  # of delta from the stored rows
    near = np.abs(ds) + p * e_out                                                                                    # |ds| with that delta
    w = (up + e) * near + p * e_dp
    m = p @ np.abs(k)
    if dtype == "bf16":
        total = w.sum(axis=1, keepdims=True)
        dq = w @ np.abs(k) + m * total + (2.0 ** -7 + 2 * e) * m * (e_out + total)
        e_delta = (e * near + p * e_dp).sum(axis=1, keepdims=True) + e * (np.abs(delta) + e_out)
    else:
        dq = (w + p * e_out) @ np.abs(k)
        e_delta = e_out
    n = (rows + 40) * F
    dk = (((up + e + n) * np.abs(ds) + p * (e_dp + e_delta)).T @ np.abs(q))
    dv = ((up + e + n) * p).T @ ao
    for name, value, bound in (("grad_q", scale * (ds @ k), scale * dq), ("grad_k", scale * (ds.T @ q), scale * dk), ("grad_v", p.T @ grad_out, dv)):
        got[name] = (value, 1.02 * (u * np.abs(value) + bound) + 1e-37)
    return got
