"""What the log probabilities' entry points refuse, and the bounds of their
scratch; none of it reaches a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from aethelstream_b200 import _lib as L
    return L


P = C.c_void_p(4096)  # a non-null, aligned address that no refused call reads
ODD = C.c_void_p(4098)
ARG, UNSUPPORTED = -1, -4


def forward(lib, hidden=P, ld_h=64, weight=P, ld_w=64, dtype=2, labels=P, n=4, d=64, v=100, top=3, lp=P, ent=P, lse=P, tv=P, ti=P,
            ws=P, size=1 << 40):
    return lib.load().aeth_token_log_probs(hidden, ld_h, weight, ld_w, dtype, labels, n, d, v, -100, top, lp, ent, lse, tv, ti, ws,
                                           size, None)


@pytest.mark.parametrize("kw,status", [
    (dict(hidden=None), ARG), (dict(weight=None), ARG), (dict(labels=None), ARG), (dict(lp=None), ARG), (dict(ent=None), ARG),
    (dict(lse=None), ARG), (dict(tv=None), ARG), (dict(ti=None), ARG), (dict(ws=None), ARG), (dict(size=16), ARG), (dict(n=-1), ARG),
    (dict(d=0), ARG), (dict(v=0), ARG), (dict(ld_h=63), ARG), (dict(ld_w=56), ARG), (dict(dtype=7), ARG), (dict(top=-1), ARG),
    (dict(top=4, v=3), ARG), (dict(top=33), UNSUPPORTED), (dict(dtype=0), UNSUPPORTED), (dict(weight=ODD), UNSUPPORTED),
    (dict(ld_w=68), UNSUPPORTED), (dict(v=1 << 31), UNSUPPORTED), (dict(n=1 << 29, v=1 << 29), UNSUPPORTED)])
def test_forward_refusals(lib, kw, status):
    assert forward(lib, **kw) == status
    assert lib.load().aeth_last_error() == status


@pytest.mark.parametrize("kw,status", [
    (dict(lse=None), ARG), (dict(ent=None), ARG), (dict(dh=None, dw=None), ARG), (dict(ld_dh=8), ARG), (dict(ld_dw=8), ARG),
    (dict(ws=None), ARG), (dict(size=16), ARG), (dict(dtype=0), UNSUPPORTED)])
def test_backward_refusals(lib, kw, status):
    a = dict(dtype=2, lse=P, ent=P, dh=P, ld_dh=64, dw=P, ld_dw=64, ws=P, size=1 << 40)
    a.update(kw)
    assert lib.load().aeth_token_log_probs_backward(P, 64, P, 64, a["dtype"], P, 4, 64, 100, -100, a["lse"], a["ent"], P, None,
                                                    a["dh"], a["ld_dh"], a["dw"], a["ld_dw"], a["ws"], a["size"], None) == status


def test_workspace_is_bounded(lib):
    """The logits that are kept take 256 MiB at most, whatever the vocabulary."""
    L, size = lib.load(), C.c_size_t()
    assert L.aeth_token_log_probs_workspace(8192, 4096, 1 << 18, 32, 0, C.byref(size)) == 0
    ranges = 8192 * ((1 << 18) // 128) * 16
    assert size.value < ranges + 8192 * (4096 * 2 + 300) + (257 << 20)
    with_none = C.c_size_t()
    assert L.aeth_token_log_probs_workspace(8192, 4096, 1 << 18, 0, 0, C.byref(with_none)) == 0
    assert with_none.value < size.value - (200 << 20)
    for bad in ((-1, 64, 100, 0), (4, 0, 100, 0), (4, 64, 0, 0), (4, 64, 100, -1)):
        assert L.aeth_token_log_probs_workspace(*bad, 0, C.byref(size)) == ARG
    assert L.aeth_token_log_probs_workspace(4, 64, 100, 33, 0, C.byref(size)) == UNSUPPORTED
    assert L.aeth_token_log_probs_workspace(4, 64, 100, 0, 1, None) == ARG


def test_python_refusals(lib):
    import aethelstream_b200 as A
    h, w, lab = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="device tensors"):
        A.token_log_probs(h, w, lab)
    r = A.TokenLogProbs(torch.zeros(4), torch.zeros(4), torch.zeros(4), None, None)
    with pytest.raises(ValueError, match="device tensors"):
        A.token_log_probs_backward(h, w, lab, r)
