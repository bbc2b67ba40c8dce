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


def rotary(lib, which="turn", **kw):
    """A call whose arguments are right but for those of kw."""
    a = dict(freq=P, rotary_dim=64, positions=P, bits=64, period=4, q=P, qt=256, qh=64, hq=4, k=P, kt=256, kh=64, hk=1, tokens=4,
             d=64, dtype=2, qg=P, kg=P, gain_dtype=2, qo=P, ko=P, dq=P, dqt=256, dk=P, dwq=P, dwk=P, ws=P, size=1 << 30, plan=True)
    a.update(kw)
    L = lib.load()
    at = (lib.RotaryPlan(a["freq"], a["rotary_dim"], 0, 1.0) if a["plan"] else None, a["positions"], a["bits"], a["period"])
    qk = (a["q"], a["qt"], a["qh"], a["hq"], a["k"], a["kt"], a["kh"], a["hk"])
    size, gains = (a["tokens"], a["d"], a["dtype"]), (a["qg"], a["kg"], a["gain_dtype"], 1e-6)
    if which == "turn":
        return L.aeth_rotary(*at, *qk, *size, 0, a["qo"], a["ko"], None)
    if which == "norm":
        return L.aeth_qk_norm_rotary(*at, *qk, *gains, *size, a["qo"], a["ko"], None)
    return L.aeth_qk_norm_rotary_backward(*at, a["dq"], a["dqt"], 64, a["dk"], 256, 64, *qk, *gains, *size, a["qo"], a["ko"],
                                          a["dwq"], a["dwk"], a["ws"], a["size"], None)


@pytest.mark.parametrize("which", ["turn", "norm", "back"])
@pytest.mark.parametrize("kw,status", [
    (dict(rotary_dim=63), ARG), (dict(rotary_dim=0), ARG), (dict(rotary_dim=66), ARG), (dict(freq=None), ARG), (dict(plan=False), ARG),
    (dict(positions=None), ARG), (dict(period=0), ARG), (dict(bits=16), ARG), (dict(q=None), ARG), (dict(k=None), ARG),
    (dict(hq=-1), ARG), (dict(hk=-1), ARG), (dict(hq=0, hk=0), ARG), (dict(qh=-64), ARG), (dict(kt=-1), ARG), (dict(qo=None), ARG),
    (dict(ko=None), ARG), (dict(tokens=-1), ARG), (dict(d=0), ARG), (dict(dtype=5), ARG), (dict(d=1025), UNSUPPORTED),
    (dict(tokens=1 << 37), UNSUPPORTED), (dict(hq=1 << 21), UNSUPPORTED)])
def test_rotary_refusals(lib, which, kw, status):
    assert rotary(lib, which, **kw) == status
    assert lib.load().aeth_last_error() == status


def test_norm_refusals(lib):
    L, size = lib.load(), C.c_size_t()
    for which in ("norm", "back"):
        for kw in (dict(qg=None), dict(kg=None), dict(gain_dtype=9)):
            assert rotary(lib, which, **kw) == ARG, (which, kw)
    for kw in (dict(dq=None), dict(dk=None), dict(dqt=-1), dict(dwq=None), dict(dwk=None), dict(ws=None), dict(size=64), dict(ws=P + 8)):
        assert rotary(lib, "back", **kw) == ARG, kw
    assert L.aeth_qk_norm_rotary_backward_workspace(64, C.byref(size)) == 0 and size.value >= 64 * 4
    assert L.aeth_qk_norm_rotary_backward_workspace(0, C.byref(size)) == ARG
    assert L.aeth_qk_norm_rotary_backward_workspace(64, None) == ARG
    assert L.aeth_qk_norm_rotary_backward_workspace(2000, C.byref(size)) == UNSUPPORTED


def test_nothing_to_do(lib):
    for which in ("turn", "norm"):
        assert rotary(lib, which, tokens=0, positions=None, q=None, k=None, qo=None, ko=None) == 0


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
