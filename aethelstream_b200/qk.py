"""Rotary positions of queries and keys, alone and behind a norm of each head.

* ``RotaryPlan``: which features of a head turn, how they pair, how fast each
  pair turns, and how that is scaled for contexts longer than training's.
* ``rotary`` / ``rotary_backward``: the rotation of q and k in one launch.
* ``qk_norm_rotary`` / ``qk_norm_rotary_backward``: RMS norm of every head of q
  and k, times a gain, and the rotation, in one pass; and its gradient.

q is (..., heads, head_dim), k (..., key heads, head_dim), with any strides that
leave a head's features side by side (views into a fused qkv product are read in
place); results are new contiguous tensors.  positions holds a whole number for
each token: the shape of q without its last two dimensions, or its last ones
where the others share them.  Everything runs on the current stream of the
tensors' device and neither synchronises nor copies to the host.  Wrong shapes,
types and devices raise ValueError; statuses of the C ABI raise AethError.
"""
from __future__ import annotations

import math

import torch

from . import _lib as L
from .galore import _DTYPES
from .training import _current_device, _elsewhere, _raw_stream, _workspace_bytes

_lib = L.load()
MAX_HEAD_DIM = 1024


class RotaryPlan:
    """Pair p of a head's first `rotary_dim` features turns by t f_p at position t,
    f_p = base^(-2 p / rotary_dim).  layout "half" pairs features p and
    p + rotary_dim / 2, "interleaved" 2 p and 2 p + 1.

    scaling stretches a context by `factor`:
      "linear"  every f_p / factor;
      "ntk"     base * factor^(rotary_dim / (rotary_dim - 2)): the fastest pair
                stays, the slowest turns 1 / factor as fast;
      "yarn"    (Peng et al. 2023) pairs that turn more than `beta_fast` times in
                `original_length` positions stay, those below `beta_slow` turn
                1 / factor as fast, between them a mixture that is linear in the
                turns; cosines and sines are multiplied by 0.1 ln(factor) + 1.
                Some programs mix linearly in the pair's index instead, between
                the pairs at the two borders; their pairs in between turn at other
                speeds, which a model trained so needs as `inv_freq`.
    `inv_freq` (rotary_dim / 2 numbers, radians a position) replaces the formula,
    `amplitude` the factor of cosines and sines."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, layout: str = "half", scaling: str = "none",
                 factor: float = 1.0, original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 amplitude: float | None = None, inv_freq=None, device=None):
        what = "RotaryPlan"
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > MAX_HEAD_DIM:
            raise ValueError(f"{what}: rotary_dim must be even, 2 to {MAX_HEAD_DIM}, got {rotary_dim}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"{what}: layout must be 'half' or 'interleaved', got {layout!r}")
        if scaling not in ("none", "linear", "ntk", "yarn"):
            raise ValueError(f"{what}: scaling must be 'none', 'linear', 'ntk' or 'yarn', got {scaling!r}")
        if not (base > 0 and math.isfinite(base) and factor > 0 and math.isfinite(factor)):
            raise ValueError(f"{what}: base and factor must be positive")
        if inv_freq is not None:
            if scaling != "none":
                raise ValueError(f"{what}: inv_freq is taken as it is; scale it beforehand")
            f = [float(x) for x in inv_freq]
            if len(f) != rotary_dim // 2:
                raise ValueError(f"{what}: inv_freq must hold {rotary_dim // 2} numbers")
        else:
            if scaling == "ntk":
                if rotary_dim == 2:
                    raise ValueError(f"{what}: 'ntk' needs two pairs at least")
                base = base * factor ** (rotary_dim / (rotary_dim - 2))
            f = [base ** (-2 * p / rotary_dim) for p in range(rotary_dim // 2)]
            if scaling == "linear":
                f = [x / factor for x in f]
            elif scaling == "yarn":
                if not original_length or original_length < 0 or not 0 <= beta_slow < beta_fast:
                    raise ValueError(f"{what}: 'yarn' needs original_length and beta_slow < beta_fast")
                for p, x in enumerate(f):
                    turns = original_length * x / math.tau
                    keep = min(max((turns - beta_slow) / (beta_fast - beta_slow), 0.0), 1.0)
                    f[p] = x * keep + x / factor * (1.0 - keep)
        if not all(math.isfinite(x) for x in f):
            raise ValueError(f"{what}: frequencies must be finite")
        if amplitude is None:
            amplitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and factor > 1.0 else 1.0
        self.rotary_dim, self.layout, self.amplitude, self.inv_freq = rotary_dim, layout, float(amplitude), tuple(f)
        turns = [round(x / math.tau * 2.0 ** 64) % 2 ** 64 for x in f]  # of 2^64 a position
        self.freq = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)
        self._c = L.RotaryPlan(self.freq.data_ptr(), rotary_dim, layout == "interleaved", self.amplitude)
        self._device = self.freq.get_device()


def _heads(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(a tensor whose data are t's head rows, the tokens' pitch, the heads'), `t`
    itself where its strides allow it."""
    shape, stride = t.shape, t.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        t = t.contiguous()
        stride = t.stride()
    if len(shape) == 3:
        return t, stride[0], stride[1]
    if len(shape) == 2:
        return t, 0, stride[0]
    ld = span = None
    for i in range(len(shape) - 3, -1, -1):  # the tokens' dimensions as one, the last first
        if shape[i] == 1:
            continue
        if ld is None:
            ld, span = stride[i], stride[i] * shape[i]
        elif stride[i] != span:
            t = t.contiguous()
            return t, t.stride(-3), t.stride(-2)
        else:
            span *= shape[i]
    return t, ld or 0, stride[-2]


def _checked(what, dev, plan, positions, q, k):
    """The arguments that every call has: ((plan, positions, bits, period), (q, its
    pitches and heads), (k, ...), (tokens, head_dim, dtype), what the pointers
    point at)."""
    if not isinstance(plan, RotaryPlan):
        raise ValueError(f"{what}: plan must be a RotaryPlan")
    shape, kind = q.shape, q.dtype
    dtype = _DTYPES.get(kind)
    if dtype is None or len(shape) < 2 or not plan.rotary_dim <= shape[-1] <= MAX_HEAD_DIM or shape[-2] == 0:
        raise ValueError(f"{what}: q must be a float tensor (..., heads, head_dim) with {plan.rotary_dim} to {MAX_HEAD_DIM} "
                         f"features a head, got {tuple(shape)}")
    lead, heads, d = shape[:-2], shape[-2], shape[-1]
    pshape, pkind = positions.shape, positions.dtype
    if pkind is not torch.int64 and pkind is not torch.int32:
        if pkind.is_floating_point or pkind.is_complex or pkind is torch.bool:
            raise ValueError(f"{what}: positions must be whole numbers")
        positions = positions.to(torch.int64)
        pkind = torch.int64
    if pshape != lead and (len(pshape) > len(lead) or lead[len(lead) - len(pshape):] != pshape):
        raise ValueError(f"{what}: positions must be {tuple(lead)} or its last dimensions, got {tuple(pshape)}")
    if plan._device != dev or positions.get_device() != dev or k is not None and k.get_device() != dev:
        raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
    if not positions.is_contiguous():
        positions = positions.contiguous()
    qr, q_t, q_h = _heads(q)
    if k is None:
        kr, side = None, (None, 0, 0, 0)
    else:
        kshape = k.shape
        if len(kshape) != len(shape) or kshape[:-2] != lead or kshape[-1] != d or kshape[-2] == 0 or k.dtype is not kind:
            raise ValueError(f"{what}: k must be (..., key heads, {d}) of q's type and tokens, got {tuple(kshape)}")
        kr, k_t, k_h = _heads(k)
        side = (kr.data_ptr(), k_t, k_h, kshape[-2])
    return ((plan._c, positions.data_ptr(), 64 if pkind is torch.int64 else 32, positions.numel() or 1),
            (qr.data_ptr(), q_t, q_h, heads), side, (q.numel() // (heads * d), d, dtype), (positions, qr, kr))


def _gains(what, dev, d, q_weight, k_weight, k):
    """(pointers and type of the weights, what they point at)"""
    if q_weight is None or (k_weight is None) != (k is None):
        raise ValueError(f"{what}: a weight for each of q and k expected")
    kind = q_weight.dtype
    for w in (q_weight, k_weight):
        if w is not None and (w.dim() != 1 or w.size(0) != d or w.dtype is not kind or kind not in _DTYPES):
            raise ValueError(f"{what}: weights must be float vectors of {d} features, of one type")
        if w is not None and w.get_device() != dev:
            raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
    qw, kw = q_weight.contiguous(), None if k_weight is None else k_weight.contiguous()
    return (qw.data_ptr(), None if kw is None else kw.data_ptr(), _DTYPES[kind]), (qw, kw)


def _results(q, k):
    """New contiguous tensors of q's and k's shapes, and where they are."""
    a = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k is None:
        return (a, None), (a.data_ptr(), None)
    b = torch.empty_like(k, memory_format=torch.contiguous_format)
    return (a, b), (a.data_ptr(), b.data_ptr())


def _turn(what, q, k, positions, plan, inverse):
    dev = q.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, _turn, what, q, k, positions, plan, inverse)
    at, qs, ks, size, keep = _checked(what, dev, plan, positions, q, k)  # noqa: F841 - keep: alive until the launch
    out, ptr = _results(q, k)
    st = _lib.aeth_rotary(*at, *qs, *ks, *size, inverse, *ptr, _raw_stream(dev))
    if st:
        L.check(st, "aeth_rotary")
    return out


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, plan: RotaryPlan):
    """(q, k) with every head turned to its token's position; k may be None."""
    return _turn("rotary", q, k, positions, plan, 0)


def rotary_backward(dq: torch.Tensor, dk: torch.Tensor | None, positions: torch.Tensor, plan: RotaryPlan):
    """The gradients of ``rotary``'s inputs from those of its outputs: turned back,
    with the plan's amplitude."""
    return _turn("rotary_backward", dq, dk, positions, plan, 1)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor, k_weight: torch.Tensor | None,
                   positions: torch.Tensor, plan: RotaryPlan, eps: float = 1e-6):
    """(q, k): x / sqrt(mean x^2 + eps) over each head's features, times the weight
    (head_dim features, a float type of its own), then turned to the position.
    Rounded once, at the end."""
    what, dev = "qk_norm_rotary", q.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, qk_norm_rotary, q, k, q_weight, k_weight, positions, plan, eps)
    at, qs, ks, size, keep = _checked(what, dev, plan, positions, q, k)  # noqa: F841
    gains, weights = _gains(what, dev, size[1], q_weight, k_weight, k)  # noqa: F841
    out, ptr = _results(q, k)
    st = _lib.aeth_qk_norm_rotary(*at, *qs, *ks, *gains, eps, *size, *ptr, _raw_stream(dev))
    if st:
        L.check(st, "aeth_qk_norm_rotary")
    return out


def qk_norm_rotary_backward(dq: torch.Tensor, dk: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor | None,
                            q_weight: torch.Tensor, k_weight: torch.Tensor | None, positions: torch.Tensor,
                            plan: RotaryPlan, eps: float = 1e-6):
    """(d_q, d_k, d_q_weight, d_k_weight) of ``qk_norm_rotary`` at its inputs q and
    k, for the gradients dq and dk of its outputs.  The weights' are float32,
    summed over tokens and heads in one fixed order."""
    what, dev = "qk_norm_rotary_backward", q.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, qk_norm_rotary_backward, dq, dk, q, k, q_weight, k_weight, positions, plan, eps)
    at, qs, ks, size, keep = _checked(what, dev, plan, positions, q, k)  # noqa: F841
    gains, weights = _gains(what, dev, size[1], q_weight, k_weight, k)  # noqa: F841
    for g, x in ((dq, q), (dk, k)):
        if (g is None) != (x is None) or g is not None and (g.shape != x.shape or g.dtype is not x.dtype):
            raise ValueError(f"{what}: gradients must have the shapes and types of q and k")
        if g is not None and g.get_device() != dev:
            raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
    gq, gq_t, gq_h = _heads(dq)
    gk, gk_t, gk_h = (None, 0, 0) if dk is None else _heads(dk)
    out, ptr = _results(q, k)
    dw_q = q.new_empty(size[1], dtype=torch.float32)
    dw_k = None if k is None else q.new_empty(size[1], dtype=torch.float32)
    room = _workspace_bytes("aeth_qk_norm_rotary_backward_workspace", dev, size[1])
    ws = q.new_empty(room, dtype=torch.uint8)
    st = _lib.aeth_qk_norm_rotary_backward(
        *at, gq.data_ptr(), gq_t, gq_h, None if gk is None else gk.data_ptr(), gk_t, gk_h, *qs, *ks, *gains, eps, *size, *ptr,
        dw_q.data_ptr(), None if dw_k is None else dw_k.data_ptr(), ws.data_ptr(), room, _raw_stream(dev))
    if st:
        L.check(st, "aeth_qk_norm_rotary_backward")
    return (*out, dw_q, dw_k)
