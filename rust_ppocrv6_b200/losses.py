"""Training losses of the recognition head: softmax cross entropy over the CTC vocabulary and
distillation from a teacher's top logits, without the [rows, classes] logits in memory.

No counterpart in the reference, which only infers. Definitions, ignored rows, layouts, types and
errors are those of include/rechead.h. Host forms take and return numpy arrays; "_device" forms
take raw CUDA pointers (e.g. torch tensors' data_ptr()), a workspace and a stream, allocate nothing
and can be captured into a CUDA graph.

  score  head_cross_entropy, head_distill             (loss, lse) under a packed head
  grad   head_cross_entropy_grad, head_distill_grad   (loss, lse, da, dw, dbias) of a training step
"""
from __future__ import annotations

import ctypes

import numpy as np

from ._lib import RH_ERR_INVALID_ARG, RecHeadError, check, load
from .head import Context, QuantizedWeight, _f32, _p, _rows, _use_bias, default_context

DTYPES = {"f32": 0, "bf16": 1}
_vp = ctypes.c_void_p


def _ptr(x: int | None):
    return _vp(x or None)


def _opt(x):
    return None if x is None else _p(x)


def _features(a, k: int, kt: bool):
    """(array, leading shape, rows, t_len) of [..., k] features, or of the [batch, k, T] layout."""
    a = _f32(a)
    if not kt:
        lead, rows = _rows(a, k)
        return a, lead, rows, 0
    if a.ndim != 3 or a.shape[1] != k:
        raise RecHeadError(RH_ERR_INVALID_ARG, f"expected [batch, {k}, T] features, got {a.shape}")
    b, _, t = a.shape
    return a, (b, t), b * t, t


def _i32(x, shape, what: str) -> np.ndarray:
    x = np.asarray(x)
    if not np.issubdtype(x.dtype, np.integer):
        raise RecHeadError(RH_ERR_INVALID_ARG, f"{what} must hold integers, got {x.dtype}")
    if x.shape != shape:
        raise RecHeadError(RH_ERR_INVALID_ARG, f"expected {what} of shape {shape}, got {x.shape}")
    if x.size and (int(x.max()) > 2 ** 31 - 1 or int(x.min()) < -2 ** 31):
        raise RecHeadError(RH_ERR_INVALID_ARG, f"{what} does not fit 32 bits")
    return np.ascontiguousarray(x, dtype=np.int32)


def _entries(top_idx, top_logits, lead):
    """A teacher's entries [..., n_top] as contiguous (int32, f32) arrays."""
    logits = _f32(top_logits)
    if logits.ndim != len(lead) + 1 or logits.shape[:-1] != lead:
        raise RecHeadError(RH_ERR_INVALID_ARG, f"expected teacher logits of shape {lead} + [n_top], got {logits.shape}")
    return _i32(top_idx, logits.shape, "teacher classes"), logits, logits.shape[-1]


def head_cross_entropy(a, qw: QuantizedWeight, target, bias=None, kt: bool = False):
    """(loss, lse) f32 of features a [..., k] (kt: [batch, k, T]) against target classes [...]
    ([batch, T]) under a packed head: loss = lse - z[target]; negative targets are ignored."""
    a, lead, rows, t_len = _features(a, qw.cols, kt)
    target = _i32(target, lead, "targets")
    if bias is not None:
        _use_bias(qw, bias)
    loss, lse = np.empty(lead, np.float32), np.empty(lead, np.float32)
    if rows:
        check(load().rh_head_cross_entropy(qw._ctx.handle, qw.handle, _p(a), rows, qw.cols, t_len, _p(target), _p(loss),
                                           _p(lse)))
    return loss, lse


def head_distill(a, qw: QuantizedWeight, top_idx, top_logits, temperature: float = 1.0, bias=None, kt: bool = False):
    """(loss, lse) f32 of a packed head against a teacher's top entries [..., n_top]."""
    a, lead, rows, t_len = _features(a, qw.cols, kt)
    idx, logits, n_top = _entries(top_idx, top_logits, lead)
    if bias is not None:
        _use_bias(qw, bias)
    loss, lse = np.empty(lead, np.float32), np.empty(lead, np.float32)
    if rows:
        check(load().rh_head_distill(qw._ctx.handle, qw.handle, _p(a), rows, qw.cols, t_len, _p(idx), _p(logits), n_top,
                                     float(temperature), _p(loss), _p(lse)))
    return loss, lse


def _grad_inputs(a, w_t, bias, row_grad, kt: bool):
    w_t = _f32(w_t)
    if w_t.ndim != 2:
        raise RecHeadError(RH_ERR_INVALID_ARG, f"expected [N, K] weight, got shape {w_t.shape}")
    n, k = w_t.shape
    a, lead, rows, t_len = _features(a, k, kt)
    if bias is not None:
        bias = _f32(bias).reshape(-1)
        if bias.size != n:
            raise RecHeadError(RH_ERR_INVALID_ARG, f"bias has {bias.size} elements but n is {n}")
    if row_grad is not None:
        row_grad = _f32(row_grad)
        if row_grad.shape != lead:
            raise RecHeadError(RH_ERR_INVALID_ARG, f"expected row_grad of shape {lead}, got {row_grad.shape}")
    out = (np.zeros(lead, np.float32), np.zeros(lead, np.float32), np.zeros_like(a), np.zeros_like(w_t),
           np.zeros(n, np.float32))
    return a, w_t, bias, row_grad, lead, rows, k, n, t_len, out


def head_cross_entropy_grad(a, w_t, target, bias=None, row_grad=None, kt: bool = False, ctx: Context | None = None):
    """(loss, lse, da, dw, dbias) f32 of a training step on features a and the weight w_t [N, K]:
    the gradients of sum(row_grad * loss) (row_grad None: of the plain sum)."""
    a, w_t, bias, row_grad, lead, rows, k, n, t_len, out = _grad_inputs(a, w_t, bias, row_grad, kt)
    target = _i32(target, lead, "targets")
    ctx = ctx or default_context()
    check(load().rh_head_cross_entropy_grad(ctx.handle, _p(a), rows, k, t_len, _p(w_t), n, _opt(bias), _p(target),
                                            _opt(row_grad), *map(_p, out)))
    return out


def head_distill_grad(a, w_t, top_idx, top_logits, temperature: float = 1.0, bias=None, row_grad=None,
                      kt: bool = False, ctx: Context | None = None):
    """head_cross_entropy_grad against a teacher's top entries [..., n_top]."""
    a, w_t, bias, row_grad, lead, rows, k, n, t_len, out = _grad_inputs(a, w_t, bias, row_grad, kt)
    idx, logits, n_top = _entries(top_idx, top_logits, lead)
    ctx = ctx or default_context()
    check(load().rh_head_distill_grad(ctx.handle, _p(a), rows, k, t_len, _p(w_t), n, _opt(bias), _p(idx), _p(logits),
                                      n_top, float(temperature), _opt(row_grad), *map(_p, out)))
    return out


def _bytes(got: int) -> int:
    if got < 0:
        raise RecHeadError(RH_ERR_INVALID_ARG, load().rh_last_error().decode("utf-8", "replace"))
    return int(got)


def _dtype(dtype: str) -> int:
    if dtype not in DTYPES:
        raise RecHeadError(RH_ERR_INVALID_ARG, f"dtype must be one of {sorted(DTYPES)}, got {dtype!r}")
    return DTYPES[dtype]


def head_loss_workspace_bytes(qw: QuantizedWeight, rows: int, slot: int = 0) -> int:
    """Workspace of the score device forms for up to `rows` rows."""
    return _bytes(load().rh_head_score_workspace_bytes(qw._ctx.handle, qw.handle, slot, rows))


def head_grad_workspace_bytes(ctx: Context, dtype: str, rows: int, k: int, n: int, n_top: int = 0,
                              slot: int = 0) -> int:
    """Workspace of the grad device forms for up to `rows` rows (n_top 0: cross entropy)."""
    dt = _dtype(dtype)
    return _bytes(load().rh_head_grad_workspace_bytes(ctx.handle, slot, dt, rows, k, n, n_top))


def head_cross_entropy_device(qw: QuantizedWeight, a_ptr: int, rows: int, target_ptr: int, loss_ptr: int, lse_ptr: int,
                              workspace_ptr: int, workspace_bytes: int, t_len: int = 0, stream: int = 0,
                              slot: int = 0) -> None:
    """rh_head_cross_entropy_device: f32 features, int32 targets; loss or lse may be 0 (not wanted)."""
    check(load().rh_head_cross_entropy_device(qw._ctx.handle, qw.handle, slot, _ptr(a_ptr), rows, t_len,
                                              _ptr(target_ptr), _ptr(loss_ptr), _ptr(lse_ptr), _ptr(workspace_ptr),
                                              workspace_bytes, _ptr(stream)))


def head_distill_device(qw: QuantizedWeight, a_ptr: int, rows: int, top_idx_ptr: int, top_logits_ptr: int, n_top: int,
                        temperature: float, loss_ptr: int, lse_ptr: int, workspace_ptr: int, workspace_bytes: int,
                        t_len: int = 0, stream: int = 0, slot: int = 0) -> None:
    """rh_head_distill_device: int32 classes and f32 logits [rows, n_top]."""
    check(load().rh_head_distill_device(qw._ctx.handle, qw.handle, slot, _ptr(a_ptr), rows, t_len, _ptr(top_idx_ptr),
                                        _ptr(top_logits_ptr), n_top, float(temperature), _ptr(loss_ptr), _ptr(lse_ptr),
                                        _ptr(workspace_ptr), workspace_bytes, _ptr(stream)))


def head_cross_entropy_grad_device(ctx: Context, dtype: str, a_ptr: int, rows: int, k: int, w_ptr: int, n: int,
                                   bias_ptr: int, target_ptr: int, row_grad_ptr: int, loss_ptr: int, lse_ptr: int,
                                   da_ptr: int, dw_ptr: int, dbias_ptr: int, workspace_ptr: int, workspace_bytes: int,
                                   t_len: int = 0, stream: int = 0, slot: int = 0) -> None:
    """rh_head_cross_entropy_grad_device. dtype ("f32" or "bf16"): of a, w, da and dw; every other
    tensor is f32, targets int32. bias, row_grad and each output may be 0."""
    dt = _dtype(dtype)
    check(load().rh_head_cross_entropy_grad_device(
        ctx.handle, slot, dt, _ptr(a_ptr), rows, k, t_len, _ptr(w_ptr), n, _ptr(bias_ptr), _ptr(target_ptr),
        _ptr(row_grad_ptr), _ptr(loss_ptr), _ptr(lse_ptr), _ptr(da_ptr), _ptr(dw_ptr), _ptr(dbias_ptr),
        _ptr(workspace_ptr), workspace_bytes, _ptr(stream)))


def head_distill_grad_device(ctx: Context, dtype: str, a_ptr: int, rows: int, k: int, w_ptr: int, n: int,
                             bias_ptr: int, top_idx_ptr: int, top_logits_ptr: int, n_top: int, temperature: float,
                             row_grad_ptr: int, loss_ptr: int, lse_ptr: int, da_ptr: int, dw_ptr: int, dbias_ptr: int,
                             workspace_ptr: int, workspace_bytes: int, t_len: int = 0, stream: int = 0,
                             slot: int = 0) -> None:
    """rh_head_distill_grad_device: head_cross_entropy_grad_device against a teacher's entries."""
    dt = _dtype(dtype)
    check(load().rh_head_distill_grad_device(
        ctx.handle, slot, dt, _ptr(a_ptr), rows, k, t_len, _ptr(w_ptr), n, _ptr(bias_ptr),
        _ptr(top_idx_ptr), _ptr(top_logits_ptr), n_top, float(temperature), _ptr(row_grad_ptr), _ptr(loss_ptr),
        _ptr(lse_ptr), _ptr(da_ptr), _ptr(dw_ptr), _ptr(dbias_ptr), _ptr(workspace_ptr), workspace_bytes,
        _ptr(stream)))
