"""AdamW over many tensors at once: the parameters that the low-rank step leaves
out (norm gains, biases, embeddings, the head).

``AdamWState`` holds the moments of a list of tensors, in 32 or in 8 bits, and
the step's count; ``adamw_step`` updates all of them in one launch (768 tensors
a launch), on the current stream of their device, without synchronising.  Count,
clip and, where wanted, learning rate lie on the device, so a captured step may be
replayed.  Wrong shapes, types and devices raise ValueError; statuses of the C ABI
raise AethError.
"""
from __future__ import annotations

from array import array
from dataclasses import dataclass
from operator import attrgetter

import torch

from . import _lib as L
from .galore import _DTYPES, AdamWConfig
from .training import _current_device, _elsewhere, _raw_stream

ADAMW_BLOCK = 2048  # elements that share a scale; a tensor's moments start on a whole block

_lib = L.load()


_data_ptr, _contiguous, _get_device = torch.Tensor.data_ptr, torch.Tensor.is_contiguous, torch.Tensor.get_device
_shape, _dtype = attrgetter("shape"), attrgetter("dtype")


def _kinds(what: str, tensors, dev: int) -> bytes:
    """The types of float tensors on `dev`."""
    try:
        kinds = bytes(map(_DTYPES.__getitem__, map(_dtype, tensors)))
    except KeyError:
        raise ValueError(f"{what}: float32, float16 or bfloat16 tensors expected") from None
    if not {dev}.issuperset(map(_get_device, tensors)):
        raise ValueError(f"{what}: all tensors must be on cuda:{dev}")
    return kinds


def _blocks(n: int) -> int:
    return -(-n // ADAMW_BLOCK)


@dataclass(slots=True)
class AdamWState:
    """Moments of a list of tensors, one tensor after the other, each from a whole
    block of 2048 elements on: m and v are float32, or int8 codes of the dynamic
    maps with one float32 scale per block (m_scales, v_scales).  master: float32
    parameters, laid out the same, that the steps are taken on (None: on the
    parameters themselves).  step: the steps taken, an int64 on the device, of
    which 40 bits count."""
    m: torch.Tensor
    v: torch.Tensor
    m_scales: torch.Tensor | None
    v_scales: torch.Tensor | None
    master: torch.Tensor | None
    step: torch.Tensor

    @classmethod
    def zeros(cls, params, bits: int = 32, master: bool = False) -> "AdamWState":
        """The state before the first step of `params` (all on one device)."""
        params = list(params)
        if bits not in (8, 32) or not params:
            raise ValueError("AdamWState: a list of tensors and 8 or 32 bits expected")
        dev = params[0].device
        total = sum(_blocks(p.numel()) for p in params)
        kind = torch.int8 if bits == 8 else torch.float32
        m, v = (torch.zeros(total * ADAMW_BLOCK, dtype=kind, device=dev) for _ in range(2))
        ms, vs = (torch.zeros(total, device=dev) if bits == 8 else None for _ in range(2))
        copy = None
        if master:
            copy, at = torch.zeros(total * ADAMW_BLOCK, device=dev), 0
            for p in params:
                copy[at:at + p.numel()] = p.detach().reshape(-1)
                at += _blocks(p.numel()) * ADAMW_BLOCK
        return cls(m, v, ms, vs, copy, torch.zeros((), dtype=torch.int64, device=dev))


def _state(what: str, s: AdamWState, dev: int) -> L.AdamwState:
    n = s.m.numel()
    bits = {torch.int8: 8, torch.float32: 32}.get(s.m.dtype)
    scales = (s.m_scales, s.v_scales)
    if bits is None or s.v.dtype != s.m.dtype or s.v.numel() != n or n % ADAMW_BLOCK or s.step.dtype != torch.int64 \
            or s.step.numel() != 1 or s.master is not None and (s.master.dtype != torch.float32 or s.master.numel() != n) \
            or bits == 8 and any(t is None or t.dtype != torch.float32 or t.numel() != n // ADAMW_BLOCK for t in scales):
        raise ValueError(f"{what}: an AdamWState with float32 moments, or int8 ones with float32 scales, expected")
    for t in (s.m, s.v, s.step, s.master, *(scales if bits == 8 else ())):
        if t is not None and (t.get_device() != dev or not t.is_contiguous()):
            raise ValueError(f"{what}: the state must be contiguous and on cuda:{dev}")
    return L.AdamwState(bits, s.m.data_ptr(), s.v.data_ptr(), *(t.data_ptr() if bits == 8 else None for t in scales),
                        None if s.master is None else s.master.data_ptr(), s.step.data_ptr(), n // ADAMW_BLOCK)


def _scalar(what: str, name: str, t, dev: int):
    if t is not None and (t.dtype != torch.float32 or t.numel() != 1 or t.get_device() != dev):
        raise ValueError(f"{what}: {name} must be one float32 on cuda:{dev}")
    return None if t is None else t.data_ptr()


def adamw_step(params, grads, state: AdamWState, config: AdamWConfig | None = None, clip: torch.Tensor | None = None,
               decay=None, lr: torch.Tensor | None = None) -> None:
    """One AdamW step of every tensor of `params` (contiguous, float32, float16 or
    bfloat16, mixed as they come), in place: with t the count of this step and
    g = clip * gradient,
      m = beta1 m + (1 - beta1) g, v = beta2 v + (1 - beta2) g^2,
      p -= lr (m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps) + weight_decay p).
    `grads`: one for each tensor, of its shape and any of the three types, and not
    in the memory of another tensor; None leaves the tensor and its moments as they
    are.  Tensors that share memory are refused where two of them have gradients.
    clip: a float32 on the device
    (what ``GaLoreOptimizer.finish_step`` leaves in its clip_out).  decay: a truth
    value for each tensor, whether weight_decay applies to it (None: to all).
    lr: a float32 on the device in config.lr's place, for a captured step."""
    what = "adamw_step"
    config = config or AdamWConfig()
    dev = state.m.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, adamw_step, params, grads, state, config, clip, decay, lr)
    params, grads = list(params), list(grads)
    count = len(params)
    if len(grads) != count or decay is not None and len(decay) != count:
        raise ValueError(f"{what}: a gradient (or None) and, where given, a decay for each of {count} tensors expected")
    if config.scale_lr_by_rank:
        raise ValueError(f"{what}: scale_lr_by_rank is for low-rank parameters")
    # by whole lists: a step of hundreds of tensors spends its host time here
    kinds = _kinds(what, params, dev)
    here, there = params, [g for g in grads if g is not None]
    some = len(there) != count
    if some:
        here = [p for p, g in zip(params, grads) if g is not None]
    gkinds = _kinds(what, there, dev)
    if not all(map(_contiguous, params)):
        raise ValueError(f"{what}: the tensors must be contiguous")
    shapes = list(map(_shape, params))
    if (list(map(_shape, here)) if some else shapes) != list(map(_shape, there)):
        raise ValueError(f"{what}: a gradient must have its tensor's shape")
    if not all(map(_contiguous, there)):
        there = [g.contiguous() for g in there]
    g_ptr = array("Q", map(_data_ptr, there))
    if some:
        left = iter(zip(g_ptr, gkinds))
        each = [(0, 0) if g is None else next(left) for g in grads]
        g_ptr, gkinds = array("Q", [x for x, _ in each]), bytes(k for _, k in each)
    p_ptr, sizes = array("Q", map(_data_ptr, params)), array("q", map(torch.Size.numel, shapes))
    blocks = sum([-(-n // ADAMW_BLOCK) for n in sizes])
    c = _state(what, state, dev)
    if blocks != c.blocks:
        raise ValueError(f"{what}: the state is for {c.blocks} blocks of {ADAMW_BLOCK} elements, the tensors have {blocks}")
    clip_ptr, lr_ptr = _scalar(what, "clip", clip, dev), _scalar(what, "lr", lr, dev)
    st = _lib.aeth_adamw_step(
        p_ptr.buffer_info()[0], g_ptr.buffer_info()[0], sizes.buffer_info()[0], kinds, gkinds,
        None if decay is None else bytes(map(bool, decay)), count, c, config.beta1, config.beta2, config.eps, config.lr,
        lr_ptr, config.weight_decay, clip_ptr, _raw_stream(dev))
    if st == L.AETH_ERR_ARG:
        raise ValueError(f"{what}: tensors that the step writes share memory")
    if st:
        L.check(st, "aeth_adamw_step")
    torch.autograd.graph.increment_version(here)  # a backward pass that saved one of them is told


def adamw_moments(state: AdamWState) -> tuple[torch.Tensor, torch.Tensor]:
    """(m, v) in float32, laid out as the state: the state's own tensors where they
    are, else what their codes stand for."""
    what, dev = "adamw_moments", state.m.get_device()
    if dev < 0 or dev != _current_device():
        return _elsewhere(what, dev, adamw_moments, state)
    c = _state(what, state, dev)
    if c.bits == 32:
        return state.m, state.v
    m, v = (torch.empty(state.m.shape, dtype=torch.float32, device=state.m.device) for _ in range(2))
    st = _lib.aeth_adamw_moments(c, m.data_ptr(), v.data_ptr(), _raw_stream(dev))
    if st:
        L.check(st, "aeth_adamw_moments")
    return m, v
