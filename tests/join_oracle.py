"""Joining a sub-layer to the residual stream and its gradients, in 64 bits (numpy), straight from the formulas."""
import numpy as np


def rms_norm(v, eps):
    return v / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)


def branch(y, live, post, gate, scale, eps):
    y = np.where(live[:, None], y, 0.0)
    b = y if post is None else rms_norm(y, eps) * post
    b = b if gate is None else np.where(live[:, None], b * gate, 0.0)
    return scale * b


def forward(x, y, live, post, gate, scale, eps):
    return x + branch(y, live, post, gate, scale, eps)


def norm_backward(v, up, eps):
    """Gradient of rms_norm(v) times `up`, with respect to v, and the largest sum of magnitudes it is made of."""
    d = v.shape[1]
    k = 1.0 / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)
    back = k ** 3 / d
    g = k * up - v * back * (v * up).sum(axis=1, keepdims=True)
    size = np.abs(k * up) + np.abs(v) * back * np.abs(v * up).sum(axis=1, keepdims=True)
    return g, size


def backward(y, out, live, post, gate, scale, following, eps, grad_out, grad_normed, gate_by_channel):
    """(gradients, magnitudes): each a dict.  A gradient's magnitude is the sum of the magnitudes of its terms, which is what
    rounding errors are relative to."""
    g, size = {}, {}
    on = live[:, None]
    D = np.zeros_like(y) if grad_out is None else grad_out.copy()
    mD = np.abs(D)
    if following is not None:
        k = 1.0 / np.sqrt((out * out).mean(axis=1, keepdims=True) + eps)
        add, m = norm_backward(out, grad_normed * following, eps)
        D, mD = D + add, mD + m
        t = np.where(on, grad_normed * out * k, 0.0)
        g["grad_next"], size["grad_next"] = t.sum(axis=0), np.abs(t).sum(axis=0)
    g["grad_x"], size["grad_x"] = D, mD
    y = np.where(on, y, 0.0)
    D, mD = np.where(on, D, 0.0), np.where(on, mD, 0.0)
    n = y if post is None else rms_norm(y, eps)
    b = n if post is None else n * post
    db, mdb = scale * D, abs(scale) * mD
    if gate is not None:
        gate = np.where(on, np.broadcast_to(gate, y.shape), 0.0)
        t, m = db * b, mdb * np.abs(b)
        g["grad_gate"], size["grad_gate"] = (t.sum(axis=0), m.sum(axis=0)) if gate_by_channel else (t, m)
        db, mdb = db * gate, mdb * np.abs(gate)
    if post is not None:
        g["grad_post"], size["grad_post"] = (db * n).sum(axis=0), (mdb * np.abs(n)).sum(axis=0)
        k = 1.0 / np.sqrt((y * y).mean(axis=1, keepdims=True) + eps)
        dy, _ = norm_backward(y, db * post, eps)
        m = mdb * np.abs(post)
        size["grad_y"] = k * m + np.abs(y) * k ** 3 / y.shape[1] * (np.abs(y) * m).sum(axis=1, keepdims=True)
        db = np.where(on, dy, 0.0)
    else:
        size["grad_y"] = mdb
    g["grad_y"] = db
    return g, size
