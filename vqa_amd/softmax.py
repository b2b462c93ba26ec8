"""Softmax read-out of rows of scores on the GPU: log probabilities of given outcomes, entropies, most probable outcomes,
and the gradient of a loss that weighs them (vqa_log_probs*, vqa_psr_chain_dev of the C ABI).

A row of scores is what a model answers with: the expectation values of its observables for one sample, one column an
outcome.  p = softmax(scale * scores) is the read-out of softmax classifiers and policies; the reference's classifier reads
class frequencies instead (vqa/QNN/myQNNs_classifier.py:1158-1269), so these functions have no counterpart there.
"""
from __future__ import annotations

import ctypes as C
from typing import Any, NamedTuple

import numpy as np

from . import _lib

_NP_CODE = {"float64": 0, "float32": 1, "float16": 3}
_codes = None


def _torch_codes():
    """torch dtype -> (VQA_DTYPE code, dtype of sums, weights and log probabilities)."""
    global _codes
    if _codes is None:
        import torch

        _codes = {torch.float64: (0, torch.float64), torch.float32: (1, torch.float32), torch.bfloat16: (2, torch.float32),
                  torch.float16: (3, torch.float32)}
    return _codes


def _is_numpy(a):
    return isinstance(a, np.ndarray) or not hasattr(a, "is_cuda")


class LogProbs(NamedTuple):
    """log_prob [R] (None without targets), entropy [R], top_log_prob [R, k], top_index [R, k] (int32, -1 where a row has
    fewer outcomes that are not masked)."""

    log_prob: Any
    entropy: Any
    top_log_prob: Any
    top_index: Any


class LogProbsGrad(NamedTuple):
    """log_prob [R] (None without targets), entropy [R], d_logits [R, V] in the scores' type."""

    log_prob: Any
    entropy: Any
    d_logits: Any


def _np_real(a, what, dtype=None):
    """An array that the library can read: of ``dtype`` (None: its own type, float64 where that is not a float that the library
    takes), in the machine's byte order."""
    a = np.asarray(a)
    if a.dtype.kind not in "fiubO":
        raise ValueError(f"{what} must be real numbers (got {a.dtype})")
    if dtype is None:
        dtype = a.dtype.newbyteorder("=") if a.dtype.name in _NP_CODE else np.float64
    return a.astype(dtype, copy=False)


def _np_rows(a, what):
    a = _np_real(a, what)
    if a.ndim != 2:
        raise ValueError(f"{what} must be [R, V]")
    return np.ascontiguousarray(a)


def _np_targets(targets, rows, width):
    t = np.asarray(targets)
    if t.shape != (rows,) or t.dtype.kind not in "iu":
        raise ValueError("targets must be integers of shape [R]")
    return np.ascontiguousarray(np.clip(t, -1, width).astype(np.int32))


def _rows(z, what):
    """(tensor whose rows are contiguous, row stride)"""
    if z.dim() != 2:
        raise ValueError(f"{what} must be [R, V]")
    if z.dtype not in _torch_codes():
        raise ValueError(f"{what} must be float64, float32, bfloat16 or float16 (got {z.dtype})")
    if not z.is_cuda:
        raise ValueError(f"{what} must be a numpy array or a cuda tensor")
    rows, width = z.shape
    if width < 1:
        raise ValueError(f"{what} must have at least one column")
    if width > 1 and z.stride(1) != 1 or rows > 1 and z.stride(0) < width:
        z = z.contiguous()
    z = z.resolve_neg()                     # (a view that torch holds negated: its memory has the other sign)
    return z, (z.stride(0) if rows > 1 else width)


def _targets(targets, z):
    import torch

    rows, width = z.shape
    t = targets if isinstance(targets, torch.Tensor) else torch.as_tensor(np.asarray(targets), device=z.device)
    if tuple(t.shape) != (rows,) or t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise ValueError("targets must be integers of shape [R]")
    if t.device != z.device:
        raise ValueError("targets must be on the scores' device")
    if t.dtype != torch.int32:
        wide = t.to(torch.int64)                  # (their own type may hold neither -1 nor the width)
        if t.dtype == torch.uint64:
            wide = torch.where(wide < 0, width, wide)                 # from 2^63 on
        t = wide.clamp(-1, width).to(torch.int32)
    return t.contiguous().resolve_neg()


def _weights(w, z, wide, what):
    """Weights of the rows in the loss: [R], or one number for all."""
    import torch

    rows = z.shape[0]
    if w is None:
        return None
    if not isinstance(w, torch.Tensor):
        w = _np_real(w, what, np.float64)
        if w.ndim == 0:                       # filled on the stream: nothing is copied from the host, also in a captured call
            return torch.full((rows,), float(w), dtype=wide, device=z.device)
        w = torch.as_tensor(w).to(z.device, wide)
    if w.dim() == 0:
        w = w.expand(rows)
    if tuple(w.shape) != (rows,):
        raise ValueError(f"{what} must have shape [R]")
    if w.device != z.device:
        raise ValueError(f"{what} must be on the scores' device")
    if w.is_complex():
        raise ValueError(f"{what} must be real numbers (got {w.dtype})")
    return w.to(wide).contiguous().resolve_neg()


_bump = None


def _written(*tensors):
    """What the library overwrote, for torch's version counters: a backward pass that saved it raises instead of taking the new
    values.  (Tensors of inference mode have no counter.)"""
    global _bump
    if _bump is None:
        from torch.autograd.graph import increment_version as _bump
    _bump([t for t in tensors if not t.is_inference()])


def _ptr(t):
    return None if t is None else t.data_ptr()


def log_probs(logits, targets=None, top_k: int = 0, scale: float = 1.0, device: int = 0) -> LogProbs:
    """Log probabilities of softmax(scale * logits), row by row: of the outcomes ``targets`` [R] (negative: none, log
    probability 0), the entropy, and the ``top_k`` most probable outcomes (equal scores by lower index; at most 64).

    A score of -inf masks its outcome.  A row with everything masked has log probability -inf and entropy 0; a row with a
    NaN or +inf, or a target beyond its outcomes, gets NaN.  Sums and results are float64 for float64 scores and float32 for
    float32, bfloat16 and float16.

    numpy scores: host-pointer path on GPU ``device``, returns numpy.  torch cuda tensors (rows may be strided): queued on
    the current torch stream of their device, returns tensors there; nothing is recorded for autograd (the gradient is
    ``log_probs_grad``)."""
    L = _lib.lib()
    top_k, scale = int(top_k), float(scale)
    if _is_numpy(logits):
        z = _np_rows(logits, "logits")
        rows, width = z.shape
        if not 0 <= top_k <= min(64, width):
            raise ValueError("top_k must be in [0, min(64, V)]")
        wide = np.float64 if z.dtype == np.float64 else np.float32
        t = None if targets is None else _np_targets(targets, rows, width)
        lp = None if t is None else np.empty(rows, wide)
        ent, top, ix = np.empty(rows, wide), np.empty((rows, top_k), wide), np.empty((rows, top_k), np.int32)
        _lib.check(L.vqa_log_probs(device, _NP_CODE[z.dtype.name], _lib.nptr(z), rows, width, width, scale, _lib.nptr(t), top_k,
                                   _lib.nptr(lp), _lib.nptr(ent), _lib.nptr(top), _lib.nptr(ix)))
        return LogProbs(lp, ent, top, ix)
    import torch

    z, stride = _rows(logits, "logits")
    rows, width = z.shape
    if not 0 <= top_k <= min(64, width):
        raise ValueError("top_k must be in [0, min(64, V)]")
    code, wide = _torch_codes()[z.dtype]
    dev = z.device
    t = None if targets is None else _targets(targets, z)
    lp = None if t is None else torch.empty(rows, dtype=wide, device=dev)
    ent = torch.empty(rows, dtype=wide, device=dev)
    top = torch.empty((rows, top_k), dtype=wide, device=dev)
    ix = torch.empty((rows, top_k), dtype=torch.int32, device=dev)
    n = L.vqa_log_probs_workspace(code, rows, width, top_k)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _lib.check(L.vqa_log_probs_dev(dev.index, _lib.current_stream(dev.index), code, z.data_ptr(), rows, width, stride,
                                   scale, _ptr(t), top_k, _ptr(ws), _ptr(lp), ent.data_ptr(), _ptr(top), _ptr(ix)))
    return LogProbs(lp, ent, top, ix)


def log_probs_grad(logits, targets, d_log_prob=None, d_entropy=None, scale: float = 1.0, out=None, device: int = 0) -> LogProbsGrad:
    """The log probabilities and entropies of ``log_probs`` with the gradient of a loss of them: ``d_log_prob`` and
    ``d_entropy`` ([R], or one number for all rows; None: 0) are the loss's derivatives by each row's log probability and
    entropy, e.g. -1 / R for a mean negative log-likelihood, minus the advantage / R for a policy gradient.

    d_logits[r, c] = scale * (d_log_prob (delta_{c, target} - p_c) - d_entropy p_c (log p_c + entropy)), in the scores'
    type; rows without a target take d_log_prob as 0, a row with everything masked has gradient 0.  ``out``: where the
    gradient goes (same shape and type, rows may be strided, not the scores themselves).  Paths as in ``log_probs``."""
    L = _lib.lib()
    scale = float(scale)
    if targets is None and d_log_prob is not None:
        raise ValueError("d_log_prob needs the targets")
    if _is_numpy(logits):
        z = _np_rows(logits, "logits")
        rows, width = z.shape
        wide = np.float64 if z.dtype == np.float64 else np.float32
        t = None if targets is None else _np_targets(targets, rows, width)
        vec = lambda w, what: None if w is None else np.ascontiguousarray(np.broadcast_to(_np_real(w, what, wide), (rows,)))
        g, h = vec(d_log_prob, "d_log_prob"), vec(d_entropy, "d_entropy")
        if out is None:
            out = np.empty_like(z)
        elif not (isinstance(out, np.ndarray) and out.shape == z.shape and out.dtype == z.dtype and out.flags.c_contiguous
                  and out.flags.writeable):
            raise ValueError("out must be a writable C-contiguous array of the scores' shape and type")
        lp = None if t is None else np.empty(rows, wide)
        ent = np.empty(rows, wide)
        _lib.check(L.vqa_log_probs_grad(device, _NP_CODE[z.dtype.name], _lib.nptr(z), rows, width, width, scale, _lib.nptr(t),
                                        _lib.nptr(g), _lib.nptr(h), _lib.nptr(lp), _lib.nptr(ent), _lib.nptr(out), width))
        return LogProbsGrad(lp, ent, out)
    import torch

    z, stride = _rows(logits, "logits")
    rows, width = z.shape
    code, wide = _torch_codes()[z.dtype]
    dev = z.device
    t = None if targets is None else _targets(targets, z)
    g, h = _weights(d_log_prob, z, wide, "d_log_prob"), _weights(d_entropy, z, wide, "d_entropy")
    given = out is not None
    if out is None:
        out = torch.empty((rows, width), dtype=z.dtype, device=dev)
    elif (tuple(out.shape) != (rows, width) or out.dtype != z.dtype or out.device != dev or width > 1 and out.stride(1) != 1
          or rows > 1 and out.stride(0) < width or out.is_neg()):
        raise ValueError("out must have the scores' shape, type and device, with contiguous rows, and not be a negated view")
    lp = None if t is None else torch.empty(rows, dtype=wide, device=dev)
    ent = torch.empty(rows, dtype=wide, device=dev)
    n = L.vqa_log_probs_workspace(code, rows, width, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _lib.check(L.vqa_log_probs_grad_dev(dev.index, _lib.current_stream(dev.index), code, z.data_ptr(), rows, width,
                                        stride, scale, _ptr(t), _ptr(g), _ptr(h), _ptr(ws), _ptr(lp), ent.data_ptr(),
                                        out.data_ptr(), out.stride(0) if rows > 1 else width))
    if given:
        _written(out)
    return LogProbsGrad(lp, ent, out)


def psr_chain(E, d_expect, factor: float = 0.5):
    """d loss / d theta [P] from a parameter-shift sweep E [B, 2P+1, n_obs] (float64 cuda tensor, as psr_full returns it)
    and the loss's derivatives d_expect [B, n_obs] by the unshifted expectation values: the sum over samples and
    observables of d_expect (E+ - E-) times ``factor`` (1/2 for the shift pi/2).  One tensor on E's device; the ranks of a
    split batch add theirs."""
    import torch

    if E.dim() != 3 or E.dtype != torch.float64 or not E.is_cuda or E.shape[1] % 2 != 1:
        raise ValueError("E must be a float64 cuda tensor [B, 2P+1, n_obs]")
    E = E.contiguous().resolve_neg()
    B, K, n_obs = E.shape
    P = (K - 1) // 2
    if tuple(d_expect.shape) != (B, n_obs) or d_expect.device != E.device or d_expect.is_complex():
        raise ValueError("d_expect must be real numbers [B, n_obs] on E's device")
    d = d_expect.to(torch.float64).contiguous().resolve_neg()
    out = torch.empty(P, dtype=torch.float64, device=E.device)
    L = _lib.lib()
    ws = torch.empty(max(int(L.vqa_psr_chain_workspace(B, max(P, 1))) // 8, 1), dtype=torch.float64, device=E.device)
    _lib.check(L.vqa_psr_chain_dev(E.device.index, _lib.current_stream(E.device.index), E.data_ptr(), B, P, n_obs,
                                   float(factor), d.data_ptr(), ws.data_ptr(), out.data_ptr()))
    return out
