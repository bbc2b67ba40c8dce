"""AdamW over many tensors against its formula.

The moments' bits are those of the formula taken one rounding at a time in fp32,
so they are compared exactly, and so are their 8-bit codes.  A parameter is
compared with the formula in 64 bits from those moments: the quotient is off by
2^-20 of itself (the approximate root and reciprocal 2^-22 each, three products),
the sum with the decay by 2^-23 of its parts, the subtraction by half a unit of
fp32, the parameter's type by half a step.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BLOCK = 2048
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def A():
    import aethelstream_b200
    return aethelstream_b200


@pytest.fixture(scope="module")
def maps():
    import ctypes as C
    from aethelstream_b200 import _lib
    out = []
    for signed in (1, 0):
        m = (C.c_float * 256)()
        _lib.load().aeth_dynamic_map(signed, m)
        out.append(np.array(m, np.float32))
    return out


def encode(x, codes):
    """(codes, scales) of blocks of x: the nearest map entry, the lower on ties."""
    x = x.reshape(-1, BLOCK)
    top = np.abs(x).max(1)
    scale = np.where(np.isfinite(top), np.where(top < 2.0 ** -126, 0, top), np.nan).astype(np.float32)
    with np.errstate(all="ignore"):
        x = np.where(scale[:, None] > 0, x * (np.float32(1) / scale)[:, None], np.float32(0)).astype(np.float32)
    at = np.clip(np.searchsorted(codes, x), 1, 255)
    at = at - 1 + ((np.abs(x - codes[at])) < np.abs(x - codes[at - 1]))
    return at.astype(np.uint8).reshape(-1), scale


def padded(tensors):
    parts = []
    for t in tensors:
        x = t.detach().float().cpu().numpy().reshape(-1)
        parts.append(np.pad(x, (0, -x.size % BLOCK)))
    return np.concatenate(parts) if parts else np.zeros(0, np.float32)


class Check:
    """The formula beside the framework's state."""

    def __init__(self, A, params, state, cfg, maps):
        self.A, self.params, self.state, self.cfg, self.maps = A, params, state, cfg, maps
        self.spans, at = [], 0
        for p in params:
            self.spans.append((at, p.numel()))
            at += -(-p.numel() // BLOCK) * BLOCK

    def step(self, grads, clip=None, decay=None, lr=None):
        A, s, c, f = self.A, self.state, self.cfg, np.float32
        m, v = (t.cpu().numpy().copy() for t in A.adamw_moments(s))
        p0 = s.master.cpu().numpy().copy() if s.master is not None else padded(self.params)
        old = [t.cpu().numpy().copy() if t is not None else None for t in (s.m, s.v, s.m_scales, s.v_scales)]
        before = [p.detach().clone() for p in self.params]
        t = int(s.step) + 1
        A.adamw_step(self.params, grads, s, c, clip=clip, decay=decay, lr=lr)
        assert int(s.step) == t
        rate = float(lr) if lr is not None else float(f(c.lr))
        live = np.zeros(m.size, bool)
        g = np.zeros(m.size, np.float32)
        wd = np.zeros(m.size)
        for i, (a, n) in enumerate(self.spans):
            if grads[i] is not None:
                live[a:a + n] = True
                g[a:a + n] = grads[i].float().cpu().numpy().reshape(-1)
                wd[a:a + n] = float(f(c.weight_decay)) * (decay is None or bool(decay[i]))
        with np.errstate(all="ignore"):
            g = g * f(1.0 if clip is None else float(clip))
            m1 = f(c.beta1) * m + f(1 - c.beta1) * g
            v1 = f(c.beta2) * v + (f(1 - c.beta2) * g) * g
            first, second = 1 / (1 - c.beta1 ** t), 1 / (1 - c.beta2 ** t)
            u = m1.astype(np.float64) * first / (np.sqrt(v1.astype(np.float64) * second) + float(f(c.eps)))
            want = p0 - rate * (u + wd * p0)
            slack = rate * (np.abs(u) * 2.0 ** -20 + (np.abs(u) + wd * np.abs(p0)) * 2.0 ** -23) + np.abs(want) * 2.0 ** -24
        # moments
        m1, v1 = np.where(live, m1, 0), np.where(live, v1, 0)
        for name, x, now, was, scale, scale_was, code in (("m", m1, s.m, old[0], s.m_scales, old[2], self.maps[0]),
                                                          ("v", v1, s.v, old[1], s.v_scales, old[3], self.maps[1])):
            now = now.cpu().numpy()
            if scale is None:
                same = np.array_equal(now[live], x[live], equal_nan=True)
                assert same, (name, np.abs(now[live] - x[live]).max())
                assert np.array_equal(now[~live], was[~live])
                continue
            q, sc = encode(x, code)
            touched = np.zeros(sc.size, bool)
            for (a, n), gr in zip(self.spans, grads):
                touched[a // BLOCK:-(-(a + n) // BLOCK)] |= gr is not None and n > 0
            got = scale.cpu().numpy()
            assert np.array_equal(got[touched], sc[touched], equal_nan=True), name
            assert np.array_equal(got[~touched], scale_was[~touched])
            rows = np.repeat(touched & np.isfinite(sc), BLOCK)
            assert np.array_equal(now.view(np.uint8)[rows], q[rows]), (name, (now.view(np.uint8)[rows] != q[rows]).sum())
            assert np.array_equal(now[np.repeat(~touched, BLOCK)], was[np.repeat(~touched, BLOCK)])
        # parameters
        for i, (a, n) in enumerate(self.spans):
            p = self.params[i].detach()
            if grads[i] is None:
                assert torch.equal(p, before[i])
                continue
            w, sl, kind = want[a:a + n], slack[a:a + n], p.dtype
            got = p.double().cpu().numpy().reshape(-1)
            ok = np.isfinite(w)
            assert np.array_equal(np.isnan(got), np.isnan(w)), i
            tol = sl + np.abs(w) * torch.finfo(kind).eps / 2 + torch.finfo(kind).tiny
            assert (np.abs(got - w)[ok] <= tol[ok]).all(), (i, kind, np.max((np.abs(got - w) / tol)[ok]))
            if s.master is not None:
                copy = s.master[a:a + n]
                assert (np.abs(copy.double().cpu().numpy() - w)[ok] <= (sl + np.finfo(np.float32).tiny)[ok]).all()
                assert torch.equal(p.reshape(-1), copy.to(kind))


def tensors(gen, sizes, kinds, scale=0.02):
    return [(scale * torch.randn(n, generator=gen, device="cuda")).to(k) for n, k in zip(sizes, kinds)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("pk", TYPES)
@pytest.mark.parametrize("gk", TYPES)
def test_steps(A, maps, bits, master, pk, gk):
    gen = torch.Generator(device="cuda").manual_seed(1)
    sizes = [1, 7, 2048, 2049, 8192, 40000, 5, 16]
    params = tensors(gen, sizes, [pk] * 8)
    params[4] = params[4].view(64, 128)
    cfg = A.AdamWConfig(beta1=0.9, beta2=0.95, eps=1e-8, lr=1e-3, weight_decay=0.1)
    state = A.AdamWState.zeros(params, bits=bits, master=master)
    c = Check(A, params, state, cfg, maps)
    for i in range(3):
        grads = [g.view(p.shape) for g, p in zip(tensors(gen, sizes, [gk] * 8, 1e-3 * (1 + i)), params)]
        c.step(grads, clip=None if i == 0 else torch.tensor(0.37, device="cuda"))


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_types_views_and_left_out(A, maps, bits):
    """Types beside one another, tensors off 16 bytes, empty ones, gradients that
    are missing or not contiguous, decay for some, a rate on the device."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(30001, generator=gen, device="cuda")
    params = [base[1:4100], base[4100:4101], (0.1 * base[5000:9999]).half()[3:], (0.1 * base[:6000]).bfloat16().view(60, 100),
              torch.empty(0, device="cuda"), torch.randn((), generator=gen, device="cuda"), (0.1 * base[:2050]).bfloat16()[1:]]
    cfg = A.AdamWConfig(lr=1e-2, weight_decay=0.01, beta2=0.999)
    state = A.AdamWState.zeros(params, bits=bits)
    c = Check(A, params, state, cfg, maps)
    for i in range(3):
        grads = [torch.randn(p.shape, generator=gen, device="cuda").to(TYPES[(i + j) % 3]) for j, p in enumerate(params)]
        grads[3] = torch.randn(100, 60, generator=gen, device="cuda").t()
        grads[i] = None
        c.step(grads, decay=[j % 2 for j in range(7)], lr=torch.tensor(3e-3 * (i + 1), device="cuda"))
    for i in range(2):
        c.step([None] * 7)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [64, 65, 256, 257, 768, 769, 1900])
def test_long_lists(A, maps, bits, count):
    """Tables of both sizes, and several launches that count one step."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    sizes = [1 + (i * 37) % 90 for i in range(count)]
    sizes[count // 2] = 5000
    params = tensors(gen, sizes, [TYPES[i % 3] for i in range(count)])
    state = A.AdamWState.zeros(params, bits=bits)
    c = Check(A, params, state, A.AdamWConfig(), maps)
    for i in range(2):
        grads = tensors(gen, sizes, [TYPES[(i + j) % 3] for j in range(count)], 1e-2)
        grads[-1] = None
        c.step(grads)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_blocks(A, maps, bits):
    """More blocks than the grid has CTAs."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    sizes = [BLOCK * 3001 + 5, 3, BLOCK * 517]
    params = tensors(gen, sizes, [torch.bfloat16] * 3)
    state = A.AdamWState.zeros(params, bits=bits)
    c = Check(A, params, state, A.AdamWConfig(lr=1e-4, weight_decay=0.1), maps)
    for _ in range(2):
        c.step(tensors(gen, sizes, [torch.bfloat16] * 3, 1e-3))


@pytest.mark.parametrize("bits", [32, 8])
def test_more_elements_than_32_bits_count(A, bits):
    """Blocks on both sides of element 2^31, and a tensor behind them: as alone."""
    n = 2 ** 31 + 3 * BLOCK + 77
    gen = torch.Generator(device="cuda").manual_seed(12)
    big, grad = (torch.empty(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    big.normal_(generator=gen)
    grad.normal_(generator=gen)
    small, small_grad = tensors(gen, [700, 700], [torch.bfloat16] * 2)
    at = 2 ** 31 - 2 * BLOCK
    alone, alone_grad = [big[at:].clone(), small.clone()], [grad[at:], small_grad]
    state, other = A.AdamWState.zeros([big, small], bits=bits), A.AdamWState.zeros(alone, bits=bits)
    for _ in range(2):
        A.adamw_step([big, small], [grad, small_grad], state)
        A.adamw_step(alone, alone_grad, other)
    assert torch.equal(big[at:], alone[0]) and torch.equal(small, alone[1])
    assert torch.equal(state.m[at:], other.m) and torch.equal(state.v[at:], other.v)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_at_the_edges(A, maps, bits):
    """Zeros, numbers whose squares vanish, the largest ones, infinities and NaN:
    what is not finite stays in its tensor (with 8 bits: in its block)."""
    sizes = [4096] * 6
    params = [torch.full((4096,), 0.5, device="cuda") for _ in sizes]
    state = A.AdamWState.zeros(params, bits=bits)
    c = Check(A, params, state, A.AdamWConfig(lr=1e-3), maps)
    grads = [torch.zeros(4096, device="cuda"), torch.full((4096,), 1e-20, device="cuda"), torch.full((4096,), 3e38, device="cuda"),
             torch.ones(4096, device="cuda"), torch.ones(4096, device="cuda"), torch.full((4096,), 2e-38, device="cuda")]
    grads[3][17] = float("nan")
    grads[4][4000] = float("inf")
    for _ in range(2):
        c.step(grads)
    assert (params[0] == 0.5).all()
    assert torch.isfinite(params[3][:17] if bits == 32 else params[3][2048:]).all()


def test_later_steps(A, maps):
    """The bias corrections of a count far on, and of one past all corrections."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    params = tensors(gen, [3000], [torch.float32])
    state = A.AdamWState.zeros(params)
    c = Check(A, params, state, A.AdamWConfig(beta2=0.9999), maps)
    for step in (0, 9, 1234, 100003, 1 << 36):
        state.step.fill_(step)
        c.step(tensors(gen, [3000], [torch.float32], 1e-3))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured(A, bits):
    """A replayed step counts, and follows the gradients, the clip and the rate."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    sizes = [5000, 33, 20000]

    def fresh():
        g = torch.Generator(device="cuda").manual_seed(7)
        p = tensors(g, sizes, [torch.bfloat16, torch.float32, torch.float16])
        return p, A.AdamWState.zeros(p, bits=bits, master=True)

    grads = tensors(gen, sizes, [torch.float32] * 3, 1e-3)
    clip, lr = torch.tensor(1.0, device="cuda"), torch.tensor(1e-3, device="cuda")
    params, state = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.adamw_step(params, grads, state, clip=clip, lr=lr)
    other, plain = fresh()
    for i in range(3):
        grads[0].mul_(1.5)
        clip.fill_(0.5 + i)
        lr.mul_(0.5)
        graph.replay()
        A.adamw_step(other, grads, plain, clip=clip, lr=lr)
    assert int(state.step) == 3
    for a, b in zip([*params, state.m, state.v, state.master], [*other, plain.m, plain.v, plain.master]):
        assert torch.equal(a, b)


def test_saved_tensors_know(A):
    """A parameter that a backward pass still needs has changed: torch says so."""
    p = torch.ones(8, device="cuda", requires_grad=True)
    y = (p * p).sum()
    A.adamw_step([p], [torch.ones(8, device="cuda")], A.AdamWState.zeros([p]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_tensor_left_out_is_not_marked(A):
    """One without a gradient is as it was, for a backward pass that saved it too."""
    p, q = (torch.ones(8, device="cuda", requires_grad=True) for _ in range(2))
    y = (q * q).sum()
    A.adamw_step([p, q], [torch.ones(8, device="cuda"), None], A.AdamWState.zeros([p, q]))
    y.backward()
    assert (q.grad == 2).all() and (p != 1).all()


def test_refusals(A):
    p, g = [torch.zeros(3000, device="cuda"), torch.zeros(7, device="cuda")], [torch.zeros(3000, device="cuda"), None]
    s = A.AdamWState.zeros(p)
    for params, grads in ((p, g[:1]), (p[:1], g[:1]), ([p[0].double(), p[1]], g), ([p[0].cpu(), p[1]], g), (p, [g[0][:5], None]),
                          (p, [g[0].int(), None]), (p, [g[0].cpu(), None]), ([torch.zeros(6000, device="cuda")[::2], p[1]], g)):
        with pytest.raises(ValueError):
            A.adamw_step(params, grads, s)
    for kw in (dict(clip=torch.tensor(1.0)), dict(clip=torch.ones(2, device="cuda")), dict(lr=torch.tensor(1, device="cuda")),
               dict(decay=[True]), dict(config=A.AdamWConfig(scale_lr_by_rank=True))):
        with pytest.raises(ValueError):
            A.adamw_step(p, g, s, **kw)
    both = A.AdamWState.zeros([p[0], p[0]])
    with pytest.raises(ValueError, match="share memory"):  # the same tensor twice
        A.adamw_step([p[0], p[0]], [g[0], g[0]], both)
    near = torch.zeros(5000, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        A.adamw_step([near[:3000], near[2999:]], [g[0], near[2999:]], A.AdamWState.zeros([near[:3000], near[2999:]]))
    for bad in (A.AdamWState(s.m.half(), s.v, None, None, None, s.step), A.AdamWState(s.m, s.v[:2048], None, None, None, s.step),
                A.AdamWState(s.m.char(), s.v.char(), None, None, None, s.step), A.AdamWState(s.m, s.v, None, None, s.m[:7], s.step),
                A.AdamWState(s.m, s.v, None, None, None, s.step.int()), A.AdamWState(s.m, s.v.cpu(), None, None, None, s.step)):
        with pytest.raises(ValueError):
            A.adamw_step(p, g, bad)
    with pytest.raises(ValueError):
        A.AdamWState.zeros(p, bits=16)
    assert int(s.step) == 0 and (p[0] == 0).all()


FIRST = """
import sys
sys.path.insert(0, {root!r})
import torch
import aethelstream_b200 as A
p, g = torch.ones(3000, device="cuda"), torch.ones(3000, device="cuda")
s = A.AdamWState.zeros([p], bits=8)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    A.adamw_step([p], [g], s)
assert int(s.step) == 0 and (p == 1).all()
graph.replay()
q = torch.ones(3000, device="cuda")
t = A.AdamWState.zeros([q], bits=8)
A.adamw_step([q], [g], t)
assert torch.equal(p, q) and (p != 1).all() and torch.equal(s.m, t.m) and torch.equal(s.m_scales, t.m_scales)
print("same")
"""


def test_first_call_inside_a_capture():
    """The maps' upload, at a device's first 8-bit step, does not end a capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]
