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
from dataclasses import dataclass

import torch

from . import _lib as L
from .galore import _DTYPES

CHECKPOINT_BLOCK = 128  # features that share a scale


def _addr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _workspace(fn: str, device, *dims) -> tuple[torch.Tensor, int]:
    size = C.c_size_t()
    L.check(getattr(L.load(), fn)(*dims, C.byref(size)), fn)
    return torch.empty(size.value, dtype=torch.uint8, device=device), size.value


def _device_of(name: str, t: torch.Tensor, *others: torch.Tensor | None) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name}: device tensors expected")
    for o in others:
        if o is not None and o.device != t.device:
            raise ValueError(f"{name}: all tensors must be on {t.device}")
    return t.device


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    """`t` as a matrix of rows whose last dimension is contiguous; a view where
    the strides allow it."""
    d = t.shape[-1]
    t = t.reshape(-1, d)
    return t if t.stride(1) == 1 and _pitch(t) >= d else t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    """Row pitch of a matrix of rows (a single row's stride says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


def _tma_rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix that TMA can read in place (16-byte aligned rows), else a copy
    with padded rows."""
    t = _rows2d(t)
    if _pitch(t) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    out = torch.empty(t.shape[0], -(-t.shape[1] // 8) * 8, dtype=t.dtype, device=t.device)[:, :t.shape[1]]
    return out.copy_(t)


# ---- head loss ----
@dataclass
class CutCrossEntropy:
    """Result of ``cut_cross_entropy``: the mean loss (a 0-dimensional tensor),
    every token's loss, and the log-sum-exp that the backward starts from."""
    loss: torch.Tensor
    losses: torch.Tensor
    lse: torch.Tensor


def _head_args(what, hidden, weight, labels):
    if weight.dim() != 2 or 0 in weight.shape or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden (..., d) and weight (vocab, d) expected, "
                         f"got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype or hidden.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: hidden and weight must both be bfloat16 or both float16")
    if labels.shape != hidden.shape[:-1] or labels.dtype.is_floating_point or labels.dtype.is_complex:
        raise ValueError(f"{what}: labels must be whole numbers of shape {tuple(hidden.shape[:-1])}")
    dev = _device_of(what, hidden, weight, labels)
    return dev, _rows2d(hidden), _tma_rows(weight), labels.reshape(-1).to(torch.int64).contiguous()


def cut_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                      ignore_index: int = -100) -> CutCrossEntropy:
    """Cross entropy of softmax(hidden @ weight.T) against `labels`, the logits
    never stored.  hidden (..., d) and weight (vocab, d) are bfloat16 or
    float16; labels (...) are whole numbers.  Tokens labelled `ignore_index`
    take no part: their loss is 0 and whatever their hidden state holds is not
    read.  A label outside the vocabulary makes its token's loss and the mean
    NaN and sets DEVERR_BAD_ARG in the device error word."""
    dev, h, w, lab = _head_args("cut_cross_entropy", hidden, weight, labels)
    n, d = h.shape
    with torch.cuda.device(dev):
        losses = torch.empty(labels.shape, dtype=torch.float32, device=dev)
        lse = torch.empty(labels.shape, dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        ws, size = _workspace("aeth_cut_ce_workspace", dev, n, d, w.shape[0], 0)
        L.check(L.load().aeth_cut_ce_forward(
            _addr(h), _pitch(h), _addr(w), _pitch(w), _DTYPES[h.dtype], _addr(lab), n, d, w.shape[0],
            ignore_index, _addr(losses), _addr(lse), _addr(loss), _addr(ws), size,
            torch.cuda.current_stream().cuda_stream), "aeth_cut_ce_forward")
    return CutCrossEntropy(loss, losses, lse)


def cut_cross_entropy_backward(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ce: CutCrossEntropy,
                               grad_losses: torch.Tensor | None = None, scale: float = 1.0, ignore_index: int = -100,
                               need_hidden: bool = True, need_weight: bool = True):
    """(d_hidden, d_weight) of ``cut_cross_entropy`` in the inputs' type; None
    where not needed (a frozen head: need_weight=False).  The gradient is that
    of scale * mean loss, or of scale * sum(grad_losses * losses) where
    `grad_losses` (float32, the shape of the labels) is given."""
    what = "cut_cross_entropy_backward"
    dev, h, w, lab = _head_args(what, hidden, weight, labels)
    n, d = h.shape
    if ce.lse.dtype != torch.float32 or ce.lse.numel() != n:
        raise ValueError(f"{what}: ce must be the result of cut_cross_entropy for these tokens")
    if grad_losses is not None and (grad_losses.dtype != torch.float32 or grad_losses.numel() != n):
        raise ValueError(f"{what}: grad_losses must be float32, one per token")
    _device_of(what, h, ce.lse, grad_losses)
    if not need_hidden and not need_weight:
        return None, None
    with torch.cuda.device(dev):
        lse = ce.lse.contiguous()
        grad = None if grad_losses is None else grad_losses.contiguous()
        dh = torch.empty(hidden.shape, dtype=h.dtype, device=dev) if need_hidden else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=dev) if need_weight else None
        ws, size = _workspace("aeth_cut_ce_workspace", dev, n, d, w.shape[0], 1)
        L.check(L.load().aeth_cut_ce_backward(
            _addr(h), _pitch(h), _addr(w), _pitch(w), _DTYPES[h.dtype], _addr(lab), n, d, w.shape[0],
            ignore_index, _addr(lse), _addr(grad), float(scale), _addr(dh), d, _addr(dw), d, _addr(ws), size,
            torch.cuda.current_stream().cuda_stream), "aeth_cut_ce_backward")
    return dh, dw


# ---- checkpointed norm ----
@dataclass
class ActivationCheckpoint:
    """Activations in 8 bits: codes (..., d) int8 and one float32 scale per row
    and block of CHECKPOINT_BLOCK features, (..., ceil(d / 128)); `dtype` is the
    type that they had and are restored to."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype


def _gain(what, gain, d):
    if gain.dim() != 1 or gain.shape[0] != d or gain.dtype not in _DTYPES:
        raise ValueError(f"{what}: weight must be a float vector of {d} features")
    return gain.contiguous()


def _ckpt_args(what, ckpt):
    codes, scales = ckpt.codes, ckpt.scales
    d = codes.shape[-1] if codes.dim() else 0
    rows = codes.numel() // d if d else 0
    blocks = -(-d // CHECKPOINT_BLOCK)
    if codes.dtype != torch.int8 or scales.dtype != torch.float32 or d == 0 or scales.numel() != rows * blocks \
            or scales.shape[-1] != blocks or ckpt.dtype not in _DTYPES:
        raise ValueError(f"{what}: an ActivationCheckpoint with int8 codes (..., d) and float32 scales "
                         f"(..., ceil(d / {CHECKPOINT_BLOCK})) expected")
    return _device_of(what, codes, scales), codes.contiguous(), scales.contiguous(), rows, d


def rms_norm_checkpoint(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                        residual: torch.Tensor | None = None):
    """RMS norm of x (..., d) times `weight`, and x in 8 bits for the second
    pass: (y, checkpoint).  With `residual` the norm's input is x + residual,
    rounded to x's type: (y, checkpoint, sum).  float32, float16 or bfloat16."""
    what = "rms_norm_checkpoint"
    if x.dtype not in _DTYPES or x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what}: x must be a float tensor (..., d)")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{what}: residual must match x")
    dev = _device_of(what, x, weight, residual)
    d = x.shape[-1]
    gain = _gain(what, weight, d)
    xr = _rows2d(x)
    rr = None if residual is None else _rows2d(residual)
    with torch.cuda.device(dev):
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        codes = torch.empty(x.shape, dtype=torch.int8, device=dev)
        scales = torch.empty((*x.shape[:-1], -(-d // CHECKPOINT_BLOCK)), dtype=torch.float32, device=dev)
        total = None if rr is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
        L.check(L.load().aeth_rms_norm_checkpoint(
            _addr(xr), _pitch(xr), _addr(rr), 0 if rr is None else _pitch(rr), _addr(gain), _DTYPES[gain.dtype],
            _DTYPES[x.dtype], xr.shape[0], d, float(eps), _addr(total), _addr(y), _addr(codes), _addr(scales),
            torch.cuda.current_stream().cuda_stream), "aeth_rms_norm_checkpoint")
    ckpt = ActivationCheckpoint(codes, scales, x.dtype)
    return (y, ckpt) if residual is None else (y, ckpt, total)


def checkpoint_decode(ckpt: ActivationCheckpoint, norm_weight: torch.Tensor | None = None,
                      eps: float = 1e-6) -> torch.Tensor:
    """The checkpoint's activations restored to their type; with `norm_weight`
    their RMS norm times it (the second pass's recomputed norm)."""
    what = "checkpoint_decode"
    dev, codes, scales, rows, d = _ckpt_args(what, ckpt)
    gain = None if norm_weight is None else _gain(what, norm_weight, d)
    _device_of(what, codes, gain)
    with torch.cuda.device(dev):
        out = torch.empty(codes.shape, dtype=ckpt.dtype, device=dev)
        L.check(L.load().aeth_checkpoint_decode(
            _addr(codes), _addr(scales), rows, d, _addr(gain), 0 if gain is None else _DTYPES[gain.dtype], float(eps),
            _addr(out), d, _DTYPES[ckpt.dtype], torch.cuda.current_stream().cuda_stream), "aeth_checkpoint_decode")
    return out


def rms_norm_checkpoint_backward(dy: torch.Tensor, ckpt: ActivationCheckpoint, weight: torch.Tensor, eps: float = 1e-6,
                                 d_residual: torch.Tensor | None = None):
    """(dx, d_weight) of the RMS norm at the restored activations, for the
    gradient dy of its output.  `d_residual`, the gradient that reaches the
    norm's input past it, is added to dx.  dx has dy's type, d_weight is
    float32 (the sum over all rows, in one fixed order)."""
    what = "rms_norm_checkpoint_backward"
    dev, codes, scales, rows, d = _ckpt_args(what, ckpt)
    gain = _gain(what, weight, d)
    if dy.shape != codes.shape or dy.dtype != ckpt.dtype:
        raise ValueError(f"{what}: dy must have the checkpoint's shape and type")
    if d_residual is not None and (d_residual.shape != dy.shape or d_residual.dtype != dy.dtype):
        raise ValueError(f"{what}: d_residual must match dy")
    _device_of(what, codes, dy, gain, d_residual)
    g = _rows2d(dy)
    r = None if d_residual is None else _rows2d(d_residual)
    with torch.cuda.device(dev):
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dev)
        dw = torch.empty(d, dtype=torch.float32, device=dev)
        ws, size = _workspace("aeth_rms_norm_checkpoint_backward_workspace", dev, rows, d)
        L.check(L.load().aeth_rms_norm_checkpoint_backward(
            _addr(g), _pitch(g), _addr(codes), _addr(scales), _addr(gain), _DTYPES[gain.dtype], _addr(r),
            0 if r is None else _pitch(r), _DTYPES[dy.dtype], rows, d, float(eps), _addr(dx), _addr(dw), _addr(ws),
            size, torch.cuda.current_stream().cuda_stream), "aeth_rms_norm_checkpoint_backward")
    return dx, dw


def checkpoint_weight_grad(dy: torch.Tensor, ckpt: ActivationCheckpoint, norm_weight: torch.Tensor | None = None,
                           eps: float = 1e-6) -> torch.Tensor:
    """Weight gradient (m, d) = dy^T X of a linear layer, dy (..., m) the gradient
    of its output, X (..., d) its input: the restored checkpoint, or with
    `norm_weight` its RMS norm times that.  bfloat16 or float16."""
    what = "checkpoint_weight_grad"
    dev, codes, scales, rows, d = _ckpt_args(what, ckpt)
    gain = None if norm_weight is None else _gain(what, norm_weight, d)
    if dy.dtype != ckpt.dtype or dy.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: dy must be bfloat16 or float16, as the checkpoint")
    if dy.dim() < 1 or dy.shape[:-1] != codes.shape[:-1] or dy.shape[-1] == 0:
        raise ValueError(f"{what}: dy must be ({', '.join(map(str, codes.shape[:-1]))}, m)")
    _device_of(what, codes, dy, gain)
    g = _tma_rows(dy)
    m = g.shape[1]
    with torch.cuda.device(dev):
        dw = torch.empty(m, d, dtype=dy.dtype, device=dev)
        ws, size = _workspace("aeth_checkpoint_weight_grad_workspace", dev, rows, m, d)
        L.check(L.load().aeth_checkpoint_weight_grad(
            _addr(g), _pitch(g), _addr(codes), _addr(scales), _addr(gain), 0 if gain is None else _DTYPES[gain.dtype],
            float(eps), _DTYPES[dy.dtype], rows, m, d, _addr(dw), d, _addr(ws), size,
            torch.cuda.current_stream().cuda_stream), "aeth_checkpoint_weight_grad")
    return dw
