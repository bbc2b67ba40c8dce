"""Training operators around the optimizer step: what makes the gradients that
``GaLoreOptimizer`` consumes.

* ``cut_cross_entropy`` / ``cut_cross_entropy_backward``: the loss at the
  language model's head and its gradient, a vocabulary piece at a time, without
  keeping the logits (streaming_cut_ce, doublepass/src/loss.rs:83-377).
* ``rms_norm_checkpoint``: RMS norm that keeps its input in 8 bits, as the first
  pass leaves it for the second; ``checkpoint_decode`` restores it (or its
  norm), ``rms_norm_checkpoint_backward`` takes the norm's gradient at it.
* ``checkpoint_weight_grad``: the weight gradient of the linear layer behind
  that norm, ready for ``GaLoreOptimizer.project_layer``.

Everything runs on the current stream of the tensors' device and neither
synchronises nor copies to the host; outputs and scratch come from torch's
allocator.  Wrong shapes, types and devices raise ValueError; statuses of the C
ABI raise AethError.
"""
from __future__ import annotations

import ctypes as C
import functools
from dataclasses import dataclass

import torch

from . import _lib as L
from .galore import _DTYPES

CHECKPOINT_BLOCK = 128  # features that share a scale

_lib = L.load()
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(fn: str, dev: int, *dims: int) -> int:
    """What `fn` asks for on `dev`, the current device: it depends on the SMs."""
    size = C.c_size_t()
    L.check(getattr(_lib, fn)(*dims, C.byref(size)), fn)
    return size.value


def _elsewhere(what: str, dev: int, f, *args):
    """f(*args) with the tensors' device current, so that its allocations, its
    stream and its launch are theirs."""
    if dev < 0:
        raise ValueError(f"{what}: device tensors expected")
    with torch.cuda.device(dev):
        return f(*args)


def _same_device(what: str, dev: int, *tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: all tensors must be on cuda:{dev}")


def _rows(t: torch.Tensor, d: int) -> tuple[torch.Tensor, int, int]:
    """`t` (..., d) as rows: (a tensor whose data are those rows, their number,
    their pitch), a view where the strides allow it."""
    if t.is_contiguous():
        return t, t.numel() // d, d
    t = t.reshape(-1, d)
    if t.stride(1) == 1 and t.size(0) > 1 and t.stride(0) >= d:
        return t, t.size(0), t.stride(0)
    return t.contiguous(), t.size(0), d


def _tma_rows(t: torch.Tensor, d: int) -> tuple[torch.Tensor, int, int]:
    """The same, 16-bit rows that TMA can read in place (16-byte aligned), else a
    copy with padded rows."""
    t, n, ld = _rows(t, d)
    if ld % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, n, ld
    ld = -(-d // 8) * 8
    out = t.new_empty((n, ld))
    out[:, :d] = t.reshape(-1, d)
    return out, n, ld


# ---- head loss ----
@dataclass(slots=True)
class CutCrossEntropy:
    """Result of ``cut_cross_entropy``: the mean loss (a 0-dimensional tensor),
    every token's loss, and the log-sum-exp that the backward starts from."""
    loss: torch.Tensor
    losses: torch.Tensor
    lse: torch.Tensor


def _head_args(what, hidden, weight, labels):
    if weight.dim() != 2 or weight.numel() == 0 or hidden.dim() < 1 or hidden.size(-1) != weight.size(1):
        raise ValueError(f"{what}: hidden (..., d) and weight (vocab, d) expected, "
                         f"got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype or hidden.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: hidden and weight must both be bfloat16 or both float16")
    if labels.shape != hidden.shape[:-1] or labels.dtype.is_floating_point or labels.dtype.is_complex:
        raise ValueError(f"{what}: labels must be whole numbers of shape {tuple(hidden.shape[:-1])}")
    _same_device(what, hidden.get_device(), weight, labels)
    return labels.to(torch.int64).contiguous()


def cut_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                      ignore_index: int = -100) -> CutCrossEntropy:
    """Cross entropy of softmax(hidden @ weight.T) against `labels`, the logits
    never stored.  hidden (..., d) and weight (vocab, d) are bfloat16 or
    float16; labels (...) are whole numbers.  Tokens labelled `ignore_index`
    take no part: their loss is 0 and whatever their hidden state holds (NaN
    too) reaches nothing.  A label outside the vocabulary makes its token's loss and the mean
    NaN and sets DEVERR_BAD_ARG in the device error word."""
    dev = hidden.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere("cut_cross_entropy", dev, cut_cross_entropy, hidden, weight, labels, ignore_index)
    lab = _head_args("cut_cross_entropy", hidden, weight, labels)
    v, d = weight.shape
    h, n, ld_h = _rows(hidden, d)
    w, _, ld_w = _tma_rows(weight, d)
    losses, lse = (lab.new_empty(labels.shape, dtype=torch.float32) for _ in range(2))
    loss = lab.new_empty((), dtype=torch.float32)
    size = _workspace_bytes("aeth_cut_ce_workspace", dev, n, d, v, 0)
    ws = lab.new_empty(size, dtype=torch.uint8)
    st = _lib.aeth_cut_ce_forward(
        h.data_ptr(), ld_h, w.data_ptr(), ld_w, _DTYPES[h.dtype], lab.data_ptr(), n, d, v, ignore_index,
        losses.data_ptr(), lse.data_ptr(), loss.data_ptr(), ws.data_ptr(), size, _raw_stream(dev))
    if st:
        L.check(st, "aeth_cut_ce_forward")
    return CutCrossEntropy(loss, losses, lse)


def cut_cross_entropy_backward(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ce: CutCrossEntropy,
                               grad_losses: torch.Tensor | None = None, scale: float = 1.0, ignore_index: int = -100,
                               need_hidden: bool = True, need_weight: bool = True):
    """(d_hidden, d_weight) of ``cut_cross_entropy`` in the inputs' type; None
    where not needed (a frozen head: need_weight=False).  The gradient is that
    of scale * mean loss, or of scale * sum(grad_losses * losses) where
    `grad_losses` (float32, the shape of the labels) is given."""
    what, dev = "cut_cross_entropy_backward", hidden.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, cut_cross_entropy_backward, hidden, weight, labels, ce, grad_losses, scale,
                          ignore_index, need_hidden, need_weight)
    lab = _head_args(what, hidden, weight, labels)
    v, d = weight.shape
    h, n, ld_h = _rows(hidden, d)
    if ce.lse.dtype != torch.float32 or ce.lse.numel() != n:
        raise ValueError(f"{what}: ce must be the result of cut_cross_entropy for these tokens")
    if grad_losses is not None and (grad_losses.dtype != torch.float32 or grad_losses.numel() != n):
        raise ValueError(f"{what}: grad_losses must be float32, one per token")
    _same_device(what, dev, ce.lse, grad_losses)
    if not need_hidden and not need_weight:
        return None, None
    w, _, ld_w = _tma_rows(weight, d)
    lse = ce.lse.contiguous()
    grad = None if grad_losses is None else grad_losses.contiguous()
    dh = h.new_empty(hidden.shape) if need_hidden else None
    dw = h.new_empty(weight.shape) if need_weight else None
    size = _workspace_bytes("aeth_cut_ce_workspace", dev, n, d, v, 1)
    ws = lab.new_empty(size, dtype=torch.uint8)
    st = _lib.aeth_cut_ce_backward(
        h.data_ptr(), ld_h, w.data_ptr(), ld_w, _DTYPES[h.dtype], lab.data_ptr(), n, d, v, ignore_index,
        lse.data_ptr(), None if grad is None else grad.data_ptr(), scale, dh.data_ptr() if need_hidden else None, d,
        dw.data_ptr() if need_weight else None, d, ws.data_ptr(), size, _raw_stream(dev))
    if st:
        L.check(st, "aeth_cut_ce_backward")
    return dh, dw


# ---- checkpointed norm ----
@dataclass(slots=True)
class ActivationCheckpoint:
    """Activations in 8 bits: codes (..., d) int8 and one float32 scale per row
    and block of CHECKPOINT_BLOCK features, (..., ceil(d / 128)); `dtype` is the
    type that they had and are restored to."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype


def _gain(what, gain, d, dev):
    dt = _DTYPES.get(gain.dtype)
    if dt is None or gain.dim() != 1 or gain.size(0) != d:
        raise ValueError(f"{what}: weight must be a float vector of {d} features")
    if gain.get_device() != dev:
        raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
    return gain.contiguous(), dt


def _ckpt_args(what, ckpt, dev):
    """(codes, scales, rows, d) of a checkpoint, contiguous."""
    codes, scales = ckpt.codes, ckpt.scales
    d = codes.size(-1) if codes.dim() else 0
    rows = codes.numel() // d if d else 0
    blocks = -(-d // CHECKPOINT_BLOCK)
    if d == 0 or codes.dtype != torch.int8 or scales.dtype != torch.float32 or scales.numel() != rows * blocks \
            or scales.dim() == 0 or scales.size(-1) != blocks or ckpt.dtype not in _DTYPES:
        raise ValueError(f"{what}: an ActivationCheckpoint with int8 codes (..., d) and float32 scales "
                         f"(..., ceil(d / {CHECKPOINT_BLOCK})) expected")
    if codes.get_device() != dev or scales.get_device() != dev:
        raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
    return codes.contiguous(), scales.contiguous(), rows, d


def rms_norm_checkpoint(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                        residual: torch.Tensor | None = None):
    """RMS norm of x (..., d) times `weight`, and x in 8 bits for the second
    pass: (y, checkpoint).  With `residual` the norm's input is x + residual,
    rounded to x's type: (y, checkpoint, sum).  float32, float16 or bfloat16."""
    what, dev = "rms_norm_checkpoint", x.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, rms_norm_checkpoint, x, weight, eps, residual)
    dt = _DTYPES.get(x.dtype)
    d = x.size(-1) if x.dim() else 0
    if dt is None or d == 0:
        raise ValueError(f"{what}: x must be a float tensor (..., d)")
    gain, gain_dt = _gain(what, weight, d, dev)
    xr, rows, ld = _rows(x, d)
    total, rr, ld_r = None, None, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"{what}: residual must match x")
        _same_device(what, dev, residual)
        rr, _, ld_r = _rows(residual, d)
        total = torch.empty_like(x, memory_format=torch.contiguous_format)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    codes = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    blocks = -(-d // CHECKPOINT_BLOCK)
    scales = x.new_empty((rows, blocks) if x.dim() == 2 else (*x.shape[:-1], blocks), dtype=torch.float32)
    st = _lib.aeth_rms_norm_checkpoint(
        xr.data_ptr(), ld, None if rr is None else rr.data_ptr(), ld_r, gain.data_ptr(), gain_dt, dt, rows, d, eps,
        None if total is None else total.data_ptr(), y.data_ptr(), codes.data_ptr(), scales.data_ptr(),
        _raw_stream(dev))
    if st:
        L.check(st, "aeth_rms_norm_checkpoint")
    ckpt = ActivationCheckpoint(codes, scales, x.dtype)
    return (y, ckpt) if residual is None else (y, ckpt, total)


def checkpoint_decode(ckpt: ActivationCheckpoint, norm_weight: torch.Tensor | None = None,
                      eps: float = 1e-6) -> torch.Tensor:
    """The checkpoint's activations restored to their type; with `norm_weight`
    their RMS norm times it (the second pass's recomputed norm)."""
    what, dev = "checkpoint_decode", ckpt.codes.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, checkpoint_decode, ckpt, norm_weight, eps)
    codes, scales, rows, d = _ckpt_args(what, ckpt, dev)
    gain, gain_dt = (None, 0) if norm_weight is None else _gain(what, norm_weight, d, dev)
    out = torch.empty_like(codes, dtype=ckpt.dtype)
    st = _lib.aeth_checkpoint_decode(codes.data_ptr(), scales.data_ptr(), rows, d,
                                     None if gain is None else gain.data_ptr(), gain_dt, eps, out.data_ptr(), d,
                                     _DTYPES[ckpt.dtype], _raw_stream(dev))
    if st:
        L.check(st, "aeth_checkpoint_decode")
    return out


def rms_norm_checkpoint_backward(dy: torch.Tensor, ckpt: ActivationCheckpoint, weight: torch.Tensor, eps: float = 1e-6,
                                 d_residual: torch.Tensor | None = None):
    """(dx, d_weight) of the RMS norm at the restored activations, for the
    gradient dy of its output.  `d_residual`, the gradient that reaches the
    norm's input past it, is added to dx.  dx has dy's type, d_weight is
    float32 (the sum over all rows, in one fixed order)."""
    what, dev = "rms_norm_checkpoint_backward", dy.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, rms_norm_checkpoint_backward, dy, ckpt, weight, eps, d_residual)
    codes, scales, rows, d = _ckpt_args(what, ckpt, dev)
    gain, gain_dt = _gain(what, weight, d, dev)
    if dy.shape != codes.shape or dy.dtype != ckpt.dtype:
        raise ValueError(f"{what}: dy must have the checkpoint's shape and type")
    if d_residual is not None:
        _same_device(what, dev, d_residual)
    g, _, ld = _rows(dy, d)
    r, ld_r = None, 0
    if d_residual is not None:
        if d_residual.shape != dy.shape or d_residual.dtype != dy.dtype:
            raise ValueError(f"{what}: d_residual must match dy")
        r, _, ld_r = _rows(d_residual, d)
    dx = torch.empty_like(dy, memory_format=torch.contiguous_format)
    dw = dy.new_empty(d, dtype=torch.float32)
    size = _workspace_bytes("aeth_rms_norm_checkpoint_backward_workspace", dev, rows, d)
    ws = dy.new_empty(size, dtype=torch.uint8)
    st = _lib.aeth_rms_norm_checkpoint_backward(
        g.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), gain.data_ptr(), gain_dt,
        None if r is None else r.data_ptr(), ld_r, _DTYPES[dy.dtype], rows, d, eps, dx.data_ptr(), dw.data_ptr(),
        ws.data_ptr(), size, _raw_stream(dev))
    if st:
        L.check(st, "aeth_rms_norm_checkpoint_backward")
    return dx, dw


def checkpoint_weight_grad(dy: torch.Tensor, ckpt: ActivationCheckpoint, norm_weight: torch.Tensor | None = None,
                           eps: float = 1e-6) -> torch.Tensor:
    """Weight gradient (m, d) = dy^T X of a linear layer, dy (..., m) the gradient
    of its output, X (..., d) its input: the restored checkpoint, or with
    `norm_weight` its RMS norm times that.  bfloat16 or float16."""
    what, dev = "checkpoint_weight_grad", dy.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, checkpoint_weight_grad, dy, ckpt, norm_weight, eps)
    codes, scales, rows, d = _ckpt_args(what, ckpt, dev)
    gain, gain_dt = (None, 0) if norm_weight is None else _gain(what, norm_weight, d, dev)
    if dy.dtype != ckpt.dtype or dy.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: dy must be bfloat16 or float16, as the checkpoint")
    m = dy.size(-1) if dy.dim() else 0
    if m == 0 or dy.shape[:-1] != codes.shape[:-1]:
        raise ValueError(f"{what}: dy must be ({', '.join(map(str, codes.shape[:-1]))}, m)")
    g, _, ld = _tma_rows(dy, m)
    dw = dy.new_empty((m, d))
    size = _workspace_bytes("aeth_checkpoint_weight_grad_workspace", dev, rows, m, d)
    ws = dy.new_empty(size, dtype=torch.uint8)
    st = _lib.aeth_checkpoint_weight_grad(
        g.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), None if gain is None else gain.data_ptr(), gain_dt, eps,
        _DTYPES[dy.dtype], rows, m, d, dw.data_ptr(), d, ws.data_ptr(), size, _raw_stream(dev))
    if st:
        L.check(st, "aeth_checkpoint_weight_grad")
    return dw
