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


def _heads(t: torch.Tensor, d: int) -> tuple[torch.Tensor, int, int]:
    """(a tensor whose data are t's head rows, the tokens' pitch, the heads'), `t`
    itself where its strides allow it."""
    if t.stride(-1) != 1 and d > 1:
        t = t.contiguous()
    if t.dim() == 3:
        return t, t.stride(0), t.stride(1)
    if t.dim() == 2:
        return t, 0, t.stride(0)
    shape, stride, ld = t.shape, t.stride(), None
    for i in range(t.dim() - 3, -1, -1):  # the tokens' dimensions as one, the last first
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


class _Call:
    """The checked arguments of a call: q and k beside further pairs of their shapes."""

    def __init__(self, what, dev, positions, plan, *pairs):
        q, k = pairs[0]
        if not isinstance(plan, RotaryPlan):
            raise ValueError(f"{what}: plan must be a RotaryPlan")
        d = q.size(-1) if q.dim() >= 2 else 0
        self.dtype = _DTYPES.get(q.dtype)
        if self.dtype is None or d == 0 or q.size(-2) == 0 or plan.rotary_dim > d or d > MAX_HEAD_DIM:
            raise ValueError(f"{what}: q must be a float tensor (..., heads, head_dim) with {plan.rotary_dim} to "
                             f"{MAX_HEAD_DIM} features a head, got {tuple(q.shape)}")
        lead = q.shape[:-2]
        if k is not None and (k.dim() != q.dim() or k.shape[:-2] != lead or k.size(-1) != d or k.dtype != q.dtype
                              or k.size(-2) == 0):
            raise ValueError(f"{what}: k must be (..., key heads, {d}) of q's type and tokens, got {tuple(k.shape)}")
        for a, b in pairs[1:]:
            for x, y in ((a, q), (b, k)):
                if (x is None) != (y is None) or x is not None and (x.shape != y.shape or x.dtype != y.dtype):
                    raise ValueError(f"{what}: gradients must have the shapes and types of q and k")
        if positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype == torch.bool:
            raise ValueError(f"{what}: positions must be whole numbers")
        if positions.dim() > len(lead) or lead[len(lead) - positions.dim():] != positions.shape:
            raise ValueError(f"{what}: positions must be {tuple(lead)} or its last dimensions, got {tuple(positions.shape)}")
        for t in (positions, plan.freq, *(t for p in pairs for t in p)):
            if t is not None and t.get_device() != dev:
                raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
        if positions.dtype not in (torch.int64, torch.int32):
            positions = positions.to(torch.int64)
        self.d = d
        self.tokens = q.numel() // (q.size(-2) * d)
        self.keep = [positions.contiguous()]  # what the pointers point at
        self.plan = L.RotaryPlan(self.keep[0].data_ptr(), 64 if positions.dtype == torch.int64 else 32,
                                 max(positions.numel(), 1), plan.freq.data_ptr(), plan.rotary_dim,
                                 plan.layout == "interleaved", plan.amplitude)
        self.sides = []
        for p in pairs:
            for t in p:
                if t is None:
                    self.sides.append(L.Heads(None, 0, 0, 0))
                    continue
                r, ld_t, ld_h = _heads(t, d)
                self.keep.append(r)
                self.sides.append(L.Heads(r.data_ptr(), ld_t, ld_h, t.size(-2)))
        self.out = [None if t is None else t.new_empty(t.shape) for t in pairs[0]]
        self.out_ptr = [None if t is None else t.data_ptr() for t in self.out]

    def gains(self, what, dev, q_weight, k_weight):
        for w, o in ((q_weight, self.out[0]), (k_weight, self.out[1])):
            if (w is None) != (o is None):
                raise ValueError(f"{what}: a weight for each of q and k expected")
            if w is not None and (w.dim() != 1 or w.size(0) != self.d or w.dtype not in _DTYPES or w.dtype != q_weight.dtype):
                raise ValueError(f"{what}: weights must be float vectors of {self.d} features, of one type")
            if w is not None and w.get_device() != dev:
                raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
        ws = [None if w is None else w.contiguous() for w in (q_weight, k_weight)]
        self.keep += ws
        return [None if w is None else w.data_ptr() for w in ws] + [_DTYPES[q_weight.dtype]]


def _turn(what, q, k, positions, plan, inverse):
    dev = q.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, _turn, what, q, k, positions, plan, inverse)
    c = _Call(what, dev, positions, plan, (q, k))
    st = _lib.aeth_rotary(c.plan, c.sides[0], c.sides[1], c.tokens, c.d, c.dtype, inverse, *c.out_ptr, _raw_stream(dev))
    if st:
        L.check(st, "aeth_rotary")
    return tuple(c.out)


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
    c = _Call(what, dev, positions, plan, (q, k))
    st = _lib.aeth_qk_norm_rotary(c.plan, c.sides[0], c.sides[1], *c.gains(what, dev, q_weight, k_weight), eps, c.tokens,
                                  c.d, c.dtype, *c.out_ptr, _raw_stream(dev))
    if st:
        L.check(st, "aeth_qk_norm_rotary")
    return tuple(c.out)


def qk_norm_rotary_backward(dq: torch.Tensor, dk: torch.Tensor | None, q: torch.Tensor, k: torch.Tensor | None,
                            q_weight: torch.Tensor, k_weight: torch.Tensor | None, positions: torch.Tensor,
                            plan: RotaryPlan, eps: float = 1e-6):
    """(d_q, d_k, d_q_weight, d_k_weight) of ``qk_norm_rotary`` at its inputs q and
    k, for the gradients dq and dk of its outputs.  The weights' are float32,
    summed over tokens and heads in one fixed order."""
    what, dev = "qk_norm_rotary_backward", q.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, qk_norm_rotary_backward, dq, dk, q, k, q_weight, k_weight, positions, plan, eps)
    c = _Call(what, dev, positions, plan, (q, k), (dq, dk))
    gains = c.gains(what, dev, q_weight, k_weight)
    dw = [None if o is None else q.new_empty(c.d, dtype=torch.float32) for o in c.out]
    size = _workspace_bytes("aeth_qk_norm_rotary_backward_workspace", dev, c.d)
    ws = q.new_empty(size, dtype=torch.uint8)
    st = _lib.aeth_qk_norm_rotary_backward(
        c.plan, c.sides[2], c.sides[3], c.sides[0], c.sides[1], *gains, eps, c.tokens, c.d, c.dtype, *c.out_ptr,
        dw[0].data_ptr(), None if dw[1] is None else dw[1].data_ptr(), ws.data_ptr(), size, _raw_stream(dev))
    if st:
        L.check(st, "aeth_qk_norm_rotary_backward")
    return (*c.out, *dw)
