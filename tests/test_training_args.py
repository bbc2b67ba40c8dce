"""What the training operators refuse, and what they do with nothing to do;
none of it reaches a GPU."""
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


def head_forward(lib, hidden=P, ld_h=64, weight=P, ld_w=64, dtype=2, labels=P, n=4, d=64, v=100, losses=P, lse=P, loss=P,
                 ws=P, size=1 << 40):
    return lib.load().aeth_cut_ce_forward(hidden, ld_h, weight, ld_w, dtype, labels, n, d, v, -100, losses, lse, loss, ws,
                                          size, None)


@pytest.mark.parametrize("kw,status", [
    (dict(hidden=None), ARG), (dict(weight=None), ARG), (dict(labels=None), ARG), (dict(loss=None), ARG),
    (dict(losses=None), ARG), (dict(lse=None), ARG), (dict(ws=None), ARG), (dict(size=16), ARG), (dict(n=-1), ARG),
    (dict(d=0), ARG), (dict(v=0), ARG), (dict(ld_h=63), ARG), (dict(ld_w=56), ARG), (dict(dtype=7), ARG),
    (dict(dtype=0), UNSUPPORTED), (dict(weight=ODD), UNSUPPORTED), (dict(ld_w=68), UNSUPPORTED),
    (dict(v=1 << 31), UNSUPPORTED), (dict(n=1 << 29, v=1 << 29), UNSUPPORTED)])
def test_head_forward_refusals(lib, kw, status):
    assert head_forward(lib, **kw) == status
    assert lib.load().aeth_last_error() == status


@pytest.mark.parametrize("kw,status", [
    (dict(lse=None), ARG), (dict(dh=None, dw=None), ARG), (dict(ld_dh=8), ARG), (dict(ld_dw=8), ARG),
    (dict(ws=None), ARG), (dict(size=16), ARG), (dict(dtype=0), UNSUPPORTED)])
def test_head_backward_refusals(lib, kw, status):
    a = dict(dtype=2, lse=P, dh=P, ld_dh=64, dw=P, ld_dw=64, ws=P, size=1 << 40)
    a.update(kw)
    assert lib.load().aeth_cut_ce_backward(P, 64, P, 64, a["dtype"], P, 4, 64, 100, -100, a["lse"], None, 1.0, a["dh"],
                                           a["ld_dh"], a["dw"], a["ld_dw"], a["ws"], a["size"], None) == status


def test_checkpoint_refusals(lib):
    L = lib.load()
    ok = [P, 64, None, 0, P, 2, 2, 4, 64, 1e-6, None, P, P, P, None]

    def store(**at):
        a = list(ok)
        for i, v in at.items():
            a[int(i[1:])] = v
        return L.aeth_rms_norm_checkpoint(*a)

    for at in (dict(_0=None), dict(_1=63), dict(_4=None), dict(_5=9), dict(_6=9), dict(_7=-1), dict(_8=0), dict(_11=None),
               dict(_12=None), dict(_13=None), dict(_2=P, _3=64), dict(_2=P, _3=8, _10=P)):
        assert store(**at) == ARG, at
    assert store(_7=1 << 31) == UNSUPPORTED
    assert L.aeth_checkpoint_decode(None, P, 4, 64, None, 0, 1e-6, P, 64, 2, None) == ARG
    assert L.aeth_checkpoint_decode(P, P, 4, 64, None, 0, 1e-6, P, 63, 2, None) == ARG
    assert L.aeth_checkpoint_decode(P, P, 4, 64, P, 5, 1e-6, P, 64, 2, None) == ARG
    assert L.aeth_rms_norm_checkpoint_backward(P, 64, P, P, P, 2, None, 0, 2, 4, 64, 1e-6, P, None, P, 1 << 40, None) == ARG
    assert L.aeth_rms_norm_checkpoint_backward(P, 64, P, P, P, 2, None, 0, 2, 4, 64, 1e-6, P, P, P, 8, None) == ARG
    assert L.aeth_rms_norm_checkpoint_backward(P, 64, P, P, P, 2, P, 8, 2, 4, 64, 1e-6, P, P, P, 1 << 40, None) == ARG
    wg = lambda **k: L.aeth_checkpoint_weight_grad(k.get("dy", P), k.get("ld", 32), P, P, None, 0, 1e-6, k.get("dt", 2), 4,  # noqa: E731
                                                   k.get("m", 32), 64, P, k.get("ldw", 64), P, k.get("size", 1 << 40), None)
    assert wg(dy=None) == ARG and wg(ld=24) == ARG and wg(m=0) == ARG and wg(ldw=56) == ARG and wg(size=8) == ARG
    assert wg(dt=0) == UNSUPPORTED and wg(dy=ODD) == UNSUPPORTED and wg(ld=36) == UNSUPPORTED


def test_nothing_to_do(lib):
    L = lib.load()
    assert L.aeth_rms_norm_checkpoint(None, 64, None, 0, P, 2, 2, 0, 64, 1e-6, None, None, None, None, None) == 0
    assert L.aeth_checkpoint_decode(None, None, 0, 64, None, 0, 1e-6, None, 64, 2, None) == 0


def test_workspace_is_bounded(lib):
    """The backward's scratch grows with the tokens, not with tokens x vocabulary:
    the piece's G takes at most 256 MiB (or one 256-entry tile of the vocabulary)."""
    size = C.c_size_t()
    L = lib.load()
    assert L.aeth_cut_ce_workspace(8192, 4096, 1 << 20, 1, C.byref(size)) == 0
    rows = 8192 * 4096 * (2 + 4)  # the gathered hidden states and the fp32 sum
    assert rows + (128 << 20) < size.value < rows + (257 << 20)
    assert L.aeth_cut_ce_workspace(8192, 4096, 1 << 20, 0, C.byref(size)) == 0
    assert size.value < 8192 * (1 << 20) * 4 / 50
    assert L.aeth_cut_ce_workspace(-1, 4096, 100, 0, C.byref(size)) == ARG
    assert L.aeth_cut_ce_workspace(1, 4096, 100, 0, None) == ARG


def test_python_refusals(lib):
    import aethelstream_b200 as A
    h, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(100, 64, dtype=torch.bfloat16)
    lab = torch.zeros(4, dtype=torch.int64)
    for bad in ((h, w[:, :32], lab), (h.float(), w.float(), lab), (h, w.half(), lab), (h, w, lab[:3]), (h, w, lab.float()),
                (h, w, lab), (h, w[:0], lab)):  # the last but one: not on a device
        with pytest.raises(ValueError):
            A.cut_cross_entropy(*bad)
    ce = A.CutCrossEntropy(torch.zeros(()), torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError):
        A.cut_cross_entropy_backward(h, w, lab, ce)
    x, g = torch.zeros(4, 64), torch.ones(64)
    for bad in ((x.int(), g), (x, g[:32]), (x, g), (x[:, :0], g[:0])):
        with pytest.raises(ValueError):
            A.rms_norm_checkpoint(*bad)
    with pytest.raises(ValueError):
        A.rms_norm_checkpoint(x, g, residual=x[:3])
    ck = A.ActivationCheckpoint(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 1), torch.bfloat16)
    for bad in (ck, A.ActivationCheckpoint(ck.codes.int(), ck.scales, ck.dtype),
                A.ActivationCheckpoint(ck.codes, torch.ones(4, 2), ck.dtype),
                A.ActivationCheckpoint(ck.codes, ck.scales, torch.float64)):
        with pytest.raises(ValueError):
            A.checkpoint_decode(bad)
        with pytest.raises(ValueError):
            A.checkpoint_weight_grad(torch.zeros(4, 32, dtype=torch.bfloat16), bad)
        with pytest.raises(ValueError):
            A.rms_norm_checkpoint_backward(torch.zeros(4, 64, dtype=torch.bfloat16), bad, g)
