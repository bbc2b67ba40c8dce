"""What the rotary, per-head norm and AdamW entry points refuse, and what they do
with nothing to do; none of it reaches a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from aethelstream_b200 import _lib as L
    return L


P = 4096  # a non-null, aligned address that no refused call reads
ARG, UNSUPPORTED = -1, -4


def plan(L, **kw):
    a = dict(positions=P, position_bits=64, period=4, freq=P, rotary_dim=64, interleaved=0, amplitude=1.0)
    a.update(kw)
    return L.RotaryPlan(*a.values())


def heads(L, **kw):
    a = dict(data=P, ld_token=256, ld_head=64, heads=4)
    a.update(kw)
    return L.Heads(*a.values())


CASES = [(dict(rotary_dim=63), {}, {}, ARG), (dict(rotary_dim=0), {}, {}, ARG), (dict(rotary_dim=66), {}, {}, ARG),
         (dict(freq=None), {}, {}, ARG), (dict(positions=None), {}, {}, ARG), (dict(period=0), {}, {}, ARG),
         (dict(position_bits=16), {}, {}, ARG), ({}, dict(data=None), {}, ARG), ({}, dict(heads=-1), {}, ARG),
         ({}, dict(ld_head=-64), {}, ARG), ({}, {}, dict(tokens=-1), ARG), ({}, {}, dict(head_dim=0), ARG),
         ({}, {}, dict(dtype=5), ARG), ({}, {}, dict(head_dim=1025), UNSUPPORTED), ({}, {}, dict(tokens=1 << 39), UNSUPPORTED),
         ({}, dict(heads=0), dict(k_heads=0), ARG), ({}, {}, dict(out=None), ARG)]


@pytest.mark.parametrize("pl,qs,more,status", CASES)
def test_rotary_refusals(lib, pl, qs, more, status):
    a = dict(tokens=4, head_dim=64, dtype=2, k_heads=1, out=P)
    a.update(more)
    q, k, p = heads(lib, **qs), heads(lib, heads=a["k_heads"]), plan(lib, **pl)
    L = lib.load()
    assert L.aeth_rotary(p, q, k, a["tokens"], a["head_dim"], a["dtype"], 0, a["out"], P, None) == status
    assert L.aeth_qk_norm_rotary(p, q, k, P, P, 2, 1e-6, a["tokens"], a["head_dim"], a["dtype"], a["out"], P, None) == status
    assert L.aeth_qk_norm_rotary_backward(p, q, k, q, k, P, P, 2, 1e-6, a["tokens"], a["head_dim"], a["dtype"], a["out"], P, P, P,
                                          P, 1 << 30, None) == status


def test_norm_refusals(lib):
    L, p, q, k = lib.load(), plan(lib), heads(lib), heads(lib, heads=1)
    assert L.aeth_qk_norm_rotary(p, q, k, None, P, 2, 1e-6, 4, 64, 2, P, P, None) == ARG
    assert L.aeth_qk_norm_rotary(p, q, k, P, None, 2, 1e-6, 4, 64, 2, P, P, None) == ARG
    assert L.aeth_qk_norm_rotary(p, q, k, P, P, 9, 1e-6, 4, 64, 2, P, P, None) == ARG
    size = C.c_size_t()
    assert L.aeth_qk_norm_rotary_backward_workspace(64, C.byref(size)) == 0 and size.value >= 64 * 4
    assert L.aeth_qk_norm_rotary_backward_workspace(0, C.byref(size)) == ARG
    assert L.aeth_qk_norm_rotary_backward_workspace(64, None) == ARG
    assert L.aeth_qk_norm_rotary_backward_workspace(2000, C.byref(size)) == UNSUPPORTED
    back = lambda **a: L.aeth_qk_norm_rotary_backward(p, a.get("dq", q), k, q, k, P, P, 2, 1e-6, 4, 64, 2, P, P, a.get("dw", P), P,  # noqa: E731
                                                      a.get("ws", P), a.get("size", 1 << 30), None)
    for bad in (dict(dq=heads(lib, heads=3)), dict(dw=None), dict(ws=None), dict(size=64), dict(ws=P + 8)):
        assert back(**bad) == ARG, bad


def test_nothing_to_do(lib):
    L, p = lib.load(), plan(lib, positions=None)
    q, k = heads(lib, data=None), heads(lib, data=None, heads=0)
    assert L.aeth_rotary(p, q, k, 0, 64, 2, 0, None, None, None) == 0
    assert L.aeth_qk_norm_rotary(p, q, k, P, None, 2, 1e-6, 0, 64, 2, None, None, None) == 0


def step(lib, p=(P, 1 << 20), n=(100, 5), g=(P, P), pd=(0, 1), gd=(0, 2), count=2, **kw):
    s = dict(bits=32, m=P, v=P, m_scales=None, v_scales=None, master=None, step=P, blocks=2)
    s.update(kw)
    return lib.load().aeth_adamw_step((C.c_void_p * 2)(*p), (C.c_void_p * 2)(*g), (C.c_int64 * 2)(*n), bytes(pd), bytes(gd), None,
                                      count, lib.AdamwState(*s.values()), 0.9, 0.999, 1e-8, 1e-3, None, 0.0, None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(p=(None, P)), ARG), (dict(n=(-1, 5)), ARG), (dict(pd=(3, 0)), ARG), (dict(gd=(0, 3)), ARG), (dict(count=-1), ARG),
    (dict(bits=16), ARG), (dict(m=None), ARG), (dict(v=None), ARG), (dict(bits=8), ARG), (dict(step=None), ARG),
    (dict(blocks=1), ARG), (dict(m=P + 4), UNSUPPORTED), (dict(master=P + 8), UNSUPPORTED), (dict(blocks=1 << 31), UNSUPPORTED),
    (dict(n=(1 << 43, 5), blocks=1 << 30), UNSUPPORTED), (dict(p=(P, P)), ARG), (dict(p=(P, P + 399)), ARG),
    (dict(p=(P + 9, P)), ARG)])
def test_adamw_refusals(lib, kw, status):
    assert step(lib, **kw) == status
    assert lib.load().aeth_last_error() == status


def test_moments_refusals(lib):
    L = lib.load()
    s = dict(bits=8, m=P, v=P, m_scales=P, v_scales=P, master=None, step=P, blocks=2)
    call = lambda m=P, v=P, **kw: L.aeth_adamw_moments(lib.AdamwState(*{**s, **kw}.values()), m, v, None)  # noqa: E731
    assert call(m=None) == ARG and call(v=None) == ARG and call(bits=32) == ARG and call(m_scales=None) == ARG
    assert call(m=P + 4) == UNSUPPORTED and call(blocks=0) == 0


def test_python_refusals(lib):
    import aethelstream_b200 as A
    for kw in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=2048), dict(layout="other"), dict(scaling="other"),
               dict(base=0.0), dict(factor=float("inf")), dict(factor=-1.0), dict(rotary_dim=2, scaling="ntk"),
               dict(scaling="yarn", factor=2.0), dict(scaling="yarn", original_length=10, beta_fast=1.0, beta_slow=2.0),
               dict(inv_freq=[1.0]), dict(inv_freq=[1.0] * 32, scaling="linear"), dict(inv_freq=[float("nan")] * 32)):
        with pytest.raises(ValueError):
            A.RotaryPlan(**{"rotary_dim": 64, **kw})
    plan = A.RotaryPlan(64)
    q, pos, w = torch.zeros(4, 2, 64), torch.arange(4), torch.ones(64)
    for f, args in ((A.rotary, (q, q)), (A.rotary_backward, (q, q)), (A.qk_norm_rotary, (q, q, w, w)),
                    (A.qk_norm_rotary_backward, (q, q, q, q, w, w))):
        with pytest.raises(ValueError, match="device tensors"):
            f(*args, pos, plan)
    p = [torch.zeros(10)]
    s = A.AdamWState.zeros(p)
    with pytest.raises(ValueError, match="device tensors"):
        A.adamw_step(p, p, s)
    with pytest.raises(ValueError, match="device tensors"):
        A.adamw_moments(s)
    for bad in (dict(params=[]), dict(params=p, bits=4)):
        with pytest.raises(ValueError):
            A.AdamWState.zeros(**bad)
