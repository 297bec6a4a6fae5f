"""Operators of a training or serving step around the layer, on device pointers (``rbmoe_join_*``, ``rbmoe_orthogonalize``,
``rbmoe_muon_step`` of include/rbmoe.h).

Calls are enqueued on the device's stream (``Device.set_stream``) without synchronisation and allocate nothing.  An argument that
is not wanted is passed as 0.  Calls on one object must not overlap in time.
"""
from __future__ import annotations

import ctypes as C

from . import _lib as L
from .moe import Device, InvalidConfig, _check


def _p(address: int):
    return address or None


def _dtype(name: str) -> int:
    if name not in ("f32", "bf16"):
        raise InvalidConfig(f"dtype must be f32 or bf16, got {name}")
    return L.DTYPES[name]


class _Operator:
    _destroy = ""

    def close(self) -> None:
        if getattr(self, "handle", None):
            getattr(self._lib, self._destroy)(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class ResidualJoin(_Operator):
    """A sub-layer's output joined to the residual stream: ``out = x + scale * gate * rmsnorm(y) * post_weight`` and, for the sub-layer
    that follows, ``normed = rmsnorm(out) * next_weight``.

    Rows are ``[rows, cols]`` of ``dtype``; weights are f32 ``[cols]``; ``gate`` is "none", "channel" (f32 ``[cols]``, a parameter) or "row"
    (``[rows, cols]`` of ``dtype``).  ``post_weight_ptr`` 0: no norm behind the sub-layer; ``next_weight_ptr`` and ``normed_ptr`` 0: no
    norm follows.  Padding rows (``valid`` byte 0) take ``y`` as zero and add nothing to the gradients of parameters."""

    _destroy = "rbmoe_join_destroy"

    def __init__(self, device: Device, cols: int, *, dtype: str = "f32", gate: str = "none"):
        if gate not in L.GATES:
            raise InvalidConfig(f"gate must be none, channel or row, got {gate}")
        self.device, self.cols, self.dtype, self.gate = device, cols, dtype, gate
        self._lib = L.load()
        h = C.c_void_p()
        _check(self._lib.rbmoe_join_create(device.handle, cols, _dtype(dtype), L.GATES[gate], C.byref(h)), device.handle)
        self.handle = h

    def forward_device(self, rows: int, x_ptr: int, y_ptr: int, out_ptr: int, normed_ptr: int = 0, *, valid_ptr: int = 0,
                       post_weight_ptr: int = 0, gate_ptr: int = 0, next_weight_ptr: int = 0, scale: float = 1.0,
                       eps: float = 1e-6) -> None:
        """``out_ptr`` may be ``x_ptr`` and ``normed_ptr`` may be ``y_ptr``."""
        _check(self._lib.rbmoe_join_forward(self.handle, rows, _p(x_ptr), _p(y_ptr), _p(valid_ptr), _p(post_weight_ptr),
                                            _p(gate_ptr), scale, _p(next_weight_ptr), eps, _p(out_ptr), _p(normed_ptr)),
               self.device.handle)

    def backward_device(self, rows: int, y_ptr: int, out_ptr: int, grad_out_ptr: int, grad_normed_ptr: int, grad_x_ptr: int,
                        grad_y_ptr: int, *, valid_ptr: int = 0, post_weight_ptr: int = 0, gate_ptr: int = 0,
                        next_weight_ptr: int = 0, scale: float = 1.0, eps: float = 1e-6, grad_post_ptr: int = 0,
                        grad_gate_ptr: int = 0, grad_next_ptr: int = 0, accumulate: bool = False) -> None:
        """Gradients of ``x`` and ``y``, and of the parameters asked for; ``out_ptr`` holds the rows that the forward wrote (0 where
        nothing follows).  ``accumulate`` adds to the parameters' gradients instead of overwriting them."""
        _check(self._lib.rbmoe_join_backward(self.handle, rows, _p(y_ptr), _p(out_ptr), _p(valid_ptr), _p(post_weight_ptr),
                                             _p(gate_ptr), scale, _p(next_weight_ptr), eps, _p(grad_out_ptr), _p(grad_normed_ptr),
                                             int(accumulate), _p(grad_x_ptr), _p(grad_y_ptr), _p(grad_post_ptr), _p(grad_gate_ptr),
                                             _p(grad_next_ptr)), self.device.handle)


class Muon(_Operator):
    """Orthogonalised updates of a stack of ``count`` weight matrices ``[rows, cols]`` (contiguous): Newton-Schulz products on the
    matrix cores at f32 accuracy, and the optimiser step around them."""

    _destroy = "rbmoe_muon_destroy"

    def __init__(self, device: Device, count: int, rows: int, cols: int):
        self.device, self.count, self.rows, self.cols = device, count, rows, cols
        self._lib = L.load()
        h = C.c_void_p()
        _check(self._lib.rbmoe_muon_create(device.handle, count, rows, cols, C.byref(h)), device.handle)
        self.handle = h

    def orthogonalize_device(self, in_ptr: int, out_ptr: int, *, dtype: str = "f32", out_dtype: str = "f32", steps: int = 5) -> None:
        """Singular values of every matrix to about one (``[0.68, 1.21]`` after five steps); ``out_ptr`` may be ``in_ptr``."""
        _check(self._lib.rbmoe_orthogonalize(self.handle, _p(in_ptr), _dtype(dtype), steps, _p(out_ptr), _dtype(out_dtype)),
               self.device.handle)

    def step_device(self, grad_ptr: int, momentum_ptr: int, weight_ptr: int, *, dtype: str = "f32", lr: float,
                    momentum: float = 0.95, weight_decay: float = 0.0, update_scale: float = 0.0, nesterov: bool = True,
                    steps: int = 5) -> None:
        """``M = momentum M + G``; ``W = (1 - lr weight_decay) W - lr update_scale O``, O the orthogonalised ``G + momentum M`` (or ``M``).
        ``dtype`` is the gradients'; M and W are f32.  ``update_scale`` 0: ``sqrt(max(1, rows / cols))``."""
        _check(self._lib.rbmoe_muon_step(self.handle, _p(grad_ptr), _dtype(dtype), _p(momentum_ptr), _p(weight_ptr), lr, momentum,
                                         weight_decay, update_scale, int(nesterov), steps), self.device.handle)
