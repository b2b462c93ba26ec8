"""Orthogonalised updates on the GPU: Newton-Schulz products that carry a matrix's singular values towards 1, and the
optimizer step around them (vqa_orthogonalize*, vqa_muon_step* of the C ABI).  For parameters that form a matrix, such as the
[layers, angles of a layer] of a layered ansatz (vqa/QNN/QML_utils.py:76-98, 143-163); ``optimizers.Muon`` steps with it.
The reference has no such optimizer.
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from . import _lib
from .softmax import _NP_CODE, _is_numpy, _np_real, _torch_codes, _written

# steepens small singular values fast; what lies in (0, 1] ends in about [0.7, 1.2] after five steps
COEFS = (3.4445, -4.7750, 2.0315)

_coefs_cache = {}


def _coefs(coefs):
    """The three coefficients as the C ABI takes them (a C array, made once for each set)."""
    key = tuple(coefs)
    got = _coefs_cache.get(key)
    if got is None:
        if len(key) != 3:
            raise ValueError("coefs are three numbers")
        if len(_coefs_cache) > 64:
            _coefs_cache.clear()
        got = _coefs_cache[key] = (C.c_double * 3)(*[float(v) for v in key])
    return got


def _matrices(g, what):
    """(tensor whose rows are contiguous, batch, rows, cols, row stride, batch stride)"""
    if g.dim() not in (2, 3):
        raise ValueError(f"{what} must be [rows, cols] or [batch, rows, cols]")
    if g.dtype not in _torch_codes():
        raise ValueError(f"{what} must be float64, float32, bfloat16 or float16 (got {g.dtype})")
    if not g.is_cuda:
        raise ValueError(f"{what} must be a numpy array or a cuda tensor")
    g = g.resolve_neg()                     # (a view that torch holds negated: its memory has the other sign)
    batch = g.shape[0] if g.dim() == 3 else 1
    rows, cols = g.shape[-2:]
    sb, sr, sc = (g.stride() if g.dim() == 3 else (0,) + tuple(g.stride()))
    if rows == 1:
        sr = cols
    if batch == 1:
        sb = rows * cols
    if cols > 1 and sc != 1 or sr < cols or batch > 1 and sb < (rows - 1) * sr + cols:
        return g.contiguous(), batch, rows, cols, cols, rows * cols
    return g, batch, rows, cols, sr, sb


def _np_matrices(g, what):
    g = _np_real(g, what)
    if g.ndim not in (2, 3):
        raise ValueError(f"{what} must be [rows, cols] or [batch, rows, cols]")
    return np.ascontiguousarray(g)


def orthogonalize(G, steps: int = 5, coefs: Sequence[float] = COEFS, eps: float = 1e-7, out=None, device: int = 0):
    """Newton-Schulz products on [rows, cols] or [batch, rows, cols]: X = G / (|G|_F + eps), then ``steps`` times
    X <- coefs[0] X + (coefs[1] A + coefs[2] A A) X with A = X X^T (on the transpose of a matrix with more rows than columns).
    The singular vectors stay, the singular values go towards 1.  Result in G's type (sums in 64 bits for float64, else 32).
    |coefs[0]| >= 1 for matrices of more than 64 rows and columns that are not float64.  A zero matrix gives zero; one with a
    NaN or inf, or whose sum of squares leaves 64 bits, gives NaN.

    numpy: host-pointer path on GPU ``device``.  torch cuda tensors (rows may be strided): queued on the current torch
    stream; ``out`` may be G itself.  Nothing is recorded for autograd; a backward pass that saved ``out`` raises."""
    L = _lib.lib()
    k = _coefs(coefs)
    if _is_numpy(G):
        g = _np_matrices(G, "G")
        batch, rows, cols = (1,) * (3 - g.ndim) + g.shape
        if out is None:
            out = np.empty_like(g)
        elif not (isinstance(out, np.ndarray) and out.shape == g.shape and out.dtype == g.dtype and out.flags.c_contiguous
                  and out.flags.writeable):
            raise ValueError("out must be a writable C-contiguous array of G's shape and type")
        _lib.check(L.vqa_orthogonalize(device, _NP_CODE[g.dtype.name], _lib.nptr(g), batch, rows, cols, cols, rows * cols, int(steps),
                                       k, float(eps), _lib.nptr(out)))
        return out
    import torch

    g, batch, rows, cols, sr, sb = _matrices(G, "G")
    code = _torch_codes()[g.dtype][0]
    dev = g.device
    given = out is not None
    if out is None:
        out = torch.empty(G.shape, dtype=g.dtype, device=dev)
    elif out.shape != G.shape or out.dtype != g.dtype or out.device != dev or not out.is_contiguous() or out.is_neg():
        raise ValueError("out must be contiguous, of G's shape, type and device, and not a negated view")
    n = L.vqa_orthogonalize_workspace(code, batch, rows, cols)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _lib.check(L.vqa_orthogonalize_dev(dev.index, _lib.current_stream(dev.index), code, g.data_ptr(), batch, rows, cols,
                                       sr, sb, int(steps), k, float(eps), None if ws is None else ws.data_ptr(), out.data_ptr()))
    if given:
        _written(out)
    return out


def muon_step(weight, grad, momentum, lr: float, mu: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True, steps: int = 5,
              coefs: Sequence[float] = COEFS, eps: float = 1e-7, device: int = 0):
    """One optimizer step on a matrix or a batch of them, in place:

        momentum <- mu * momentum + grad;  u = grad + mu * momentum  (``nesterov``)  or  momentum
        weight   <- (1 - lr * weight_decay) * weight - lr * sqrt(max(1, rows / cols)) * orthogonalize(u)

    weight and momentum are contiguous: float64 with float64 gradients, float32 with float32, bfloat16 and float16 ones.
    Returns weight.  Nothing is recorded for autograd; a backward pass that saved what is overwritten raises.  Paths as in
    ``orthogonalize`` (numpy: weight and momentum are overwritten, grad is taken in their type)."""
    L = _lib.lib()
    k = _coefs(coefs)
    if _is_numpy(weight):
        for a, what in ((weight, "weight"), (momentum, "momentum")):
            if not (isinstance(a, np.ndarray) and a.dtype in (np.float64, np.float32) and a.flags.c_contiguous and a.flags.writeable
                    and a.ndim in (2, 3)):
                raise ValueError(f"{what} must be a writable C-contiguous float64 or float32 array [rows, cols] or [batch, rows, cols]")
        g = np.ascontiguousarray(_np_real(grad, "grad", weight.dtype))
        if momentum.shape != weight.shape or momentum.dtype != weight.dtype or g.shape != weight.shape:
            raise ValueError("weight, grad and momentum must have one shape, weight and momentum one type")
        batch, rows, cols = (1,) * (3 - g.ndim) + g.shape
        _lib.check(L.vqa_muon_step(device, _NP_CODE[g.dtype.name], _lib.nptr(weight), _lib.nptr(g), _lib.nptr(momentum), batch, rows,
                                   cols, cols, rows * cols, float(lr), float(mu), float(weight_decay), int(bool(nesterov)), int(steps),
                                   k, float(eps)))
        return weight
    import torch

    g, batch, rows, cols, sr, sb = _matrices(grad, "grad")
    code, wide = _torch_codes()[g.dtype]
    dev = g.device
    for a, what in ((weight, "weight"), (momentum, "momentum")):
        if a.shape != grad.shape or a.dtype != wide or a.device != dev or not a.is_contiguous() or a.is_neg():
            raise ValueError(f"{what} must be a contiguous {wide} tensor of grad's shape on its device, and not a negated view")
    n = L.vqa_orthogonalize_workspace(code, batch, rows, cols)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _lib.check(L.vqa_muon_step_dev(dev.index, _lib.current_stream(dev.index), code, weight.data_ptr(), g.data_ptr(),
                                   momentum.data_ptr(), batch, rows, cols, sr, sb, float(lr), float(mu), float(weight_decay),
                                   int(bool(nesterov)), int(steps), k, float(eps), None if ws is None else ws.data_ptr()))
    _written(weight, momentum)
    return weight
