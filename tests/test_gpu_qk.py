"""Rotary positions and per-head norms of queries and keys against their
formulas in 64 bits.

Tolerances.  u is half a unit of fp32, 2^-24.  A cosine or sine is off by less
than 4 u (its own rounding, the angle's 3e-8, the product with the amplitude), so
a turned feature by (|u|+|v|) a (4 u + 2 u for the products and the sum) at most:
TURN = 8 u.  The norm's factor r is off by (D / 2 + 4) u of itself (D squares
added up, halved by the root; the root itself 2 u), the products with it by 2 u.
The result's own rounding is half a step of its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TURN = 8 * U
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def A():
    import aethelstream_b200
    return aethelstream_b200


def angles(plan, positions):
    """Cosines and sines (tokens..., 1, pairs) of whole positions, in 64 bits."""
    f = torch.tensor(plan.inv_freq, dtype=torch.float64, device="cuda")
    t = positions.double()[..., None, None] * f
    return plan.amplitude * torch.cos(t), plan.amplitude * torch.sin(t)


def split(plan, x):
    r = plan.rotary_dim
    if plan.layout == "half":
        return x[..., :r // 2], x[..., r // 2:r], x[..., r:]
    return x[..., :r:2], x[..., 1:r:2], x[..., r:]


def join(plan, u, v, rest):
    if plan.layout == "half":
        return torch.cat([u, v, rest], -1)
    return torch.cat([torch.stack([u, v], -1).flatten(-2), rest], -1)


def turn(plan, x, positions, sign=1.0):
    """(turned x, the bound of its error) of x in 64 bits."""
    c, s = angles(plan, positions)
    u, v, rest = split(plan, x)
    size = (u.abs() + v.abs()) * abs(plan.amplitude) * TURN
    return (join(plan, u * c - sign * v * s, v * c + sign * u * s, rest), join(plan, size, size, torch.zeros_like(rest)))


def close(got, want, slack, name=""):
    tol = slack + want.abs() * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs() - tol
    assert got.shape == want.shape and torch.isfinite(got).all() and (off <= 0).all(), (name, float(off.max()), int((off > 0).sum()))


def rows(gen, shape, dtype, how):
    """Heads as they come: whole, side by side with others, or off 16 bytes."""
    *lead, h, d = shape
    if how == "whole":
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)
    if how == "fused":
        return torch.randn((*lead, h + 3, d), generator=gen, device="cuda").to(dtype)[..., 2:2 + h, :]
    if how == "turned":  # heads before tokens
        return torch.randn((h, *lead, d), generator=gen, device="cuda").to(dtype).movedim(0, -2)
    return torch.randn((*lead, h, d + 3), generator=gen, device="cuda").to(dtype)[..., 1:1 + d]


SHAPES = [  # tokens, heads of q and k, features, those that turn
    (1, 1, 1, 2, 2), (1, 64, 8, 128, 128), (3, 5, 1, 16, 16), (77, 8, 2, 128, 128), (33, 3, 1, 96, 64), (65, 4, 4, 80, 80),
    (21, 6, 2, 80, 40), (130, 2, 1, 64, 32), (9, 3, 2, 18, 6), (12, 2, 1, 256, 256), (7, 2, 1, 512, 128), (5, 1, 1, 1024, 1024),
    (6, 2, 1, 513, 512), (700, 1, 1, 32, 32), (4, 71, 1, 192, 96),
    (9, 3, 2, 33, 32), (11, 2, 1, 129, 2), (50, 2, 3, 255, 250), (13, 4, 1, 256, 24)]


@pytest.mark.parametrize("how", ["whole", "fused", "off"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
def test_rotary(A, dtype, layout, how):
    gen = torch.Generator(device="cuda").manual_seed(1)
    for n, hq, hk, d, r in SHAPES:
        plan = A.RotaryPlan(r, layout=layout, device="cuda")
        pos = torch.randint(0, 1 << 20, (n,), generator=gen, device="cuda")
        q, k = rows(gen, (n, hq, d), dtype, how), rows(gen, (n, hk, d), dtype, how)
        for f, sign in ((A.rotary, 1.0), (A.rotary_backward, -1.0)):
            for got, x in zip(f(q, k, pos, plan), (q, k)):
                assert got.is_contiguous() and got.dtype == dtype
                close(got, *turn(plan, x.double(), pos, sign), (n, hq, d, r))


def norm(x, w, eps):
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return x * r * w, r


@pytest.mark.parametrize("how", ["whole", "fused", "off"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_and_its_gradient(A, dtype, layout, how):
    gen = torch.Generator(device="cuda").manual_seed(2)
    eps = 1e-6
    for i, (n, hq, hk, d, r) in enumerate(SHAPES):
        plan = A.RotaryPlan(r, layout=layout, scaling="yarn", factor=4.0, original_length=4096, device="cuda")
        pos = torch.randint(0, 1 << 17, (n,), generator=gen, device="cuda")
        q, k = rows(gen, (n, hq, d), dtype, how), rows(gen, (n, hk, d), dtype, how)
        wt = TYPES[i % 3]  # of the weights, a type of its own
        wq, wk = ((1 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(wt) for _ in range(2))
        dq, dk = rows(gen, (n, hq, d), dtype, how), rows(gen, (n, hk, d), dtype, how)
        factor = (d / 2 + 8) * U
        for got, x, w in zip(A.qk_norm_rotary(q, k, wq, wk, pos, plan, eps=eps), (q, k), (wq, wk)):
            y, _ = norm(x.double(), w.double(), eps)
            want, slack = turn(plan, y, pos)
            _, more = turn(plan, y, pos)  # |u|+|v| of a pair, whose relative error is `factor`
            u, v, rest = split(plan, y.abs())
            pair = join(plan, u + v, u + v, rest) * max(1.0, plan.amplitude)
            close(got, want, slack + factor * pair, ("forward", n, hq, d, r))
        got = A.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, pos, plan, eps=eps)
        for x, w, dy, dx, dw in ((q, wq, dq, got[0], got[2]), (k, wk, dk, got[1], got[3])):
            x, w = x.double(), w.double()
            g, gs = turn(plan, dy.double(), pos, -1.0)
            _, rr = norm(x, w, eps)
            mean = (w * g * x).mean(-1, keepdim=True)
            want = rr * w * g - x * rr ** 3 * mean
            slack = rr * w.abs() * gs + x.abs() * rr ** 3 * (w.abs() * gs * x.abs()).mean(-1, keepdim=True)
            # the mean's d products and r^3
            slack = slack + 4 * (d + 16) * U * ((rr * w * g).abs() + x.abs() * rr ** 3 * (w * g * x).abs().mean(-1, keepdim=True))
            close(dx, want, slack, ("dx", n, hq, d, r))
            heads = x.shape[0] * x.shape[1]
            terms = g * x * rr
            ws = (gs * (x * rr).abs()).sum((0, 1)) + (heads + d + 16) * U * terms.abs().sum((0, 1))
            assert dw.dtype == torch.float32 and dw.shape == (d,)
            close(dw, terms.sum((0, 1)), ws, ("dw", n, hq, d, r))


def test_gradient_against_differences(A):
    """d of sum(y * c) along a direction, from values a small step apart."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    n, h, d = 5, 3, 64
    plan = A.RotaryPlan(32, device="cuda")
    pos = torch.arange(n, device="cuda")
    x, c, z = (torch.randn(n, h, d, generator=gen, device="cuda") for _ in range(3))
    w = 1 + 0.1 * torch.randn(d, generator=gen, device="cuda")
    dx, _, dw, _ = A.qk_norm_rotary_backward(c, None, x, None, w, None, pos, plan)

    def value(x, w):
        y, _ = A.qk_norm_rotary(x, None, w, None, pos, plan)
        return (y.double() * c.double()).sum().item()

    # values of some 30 in fp32, 960 terms off by 2^-22 each: 2e-5 at most, over 2 * step; the third derivative's
    # part is of the size of step^2
    step = 2.0 ** -7
    slope = (value(x + step * z, w) - value(x - step * z, w)) / (2 * step)
    assert abs(slope - (dx.double() * z.double()).sum().item()) < 2e-5 * 30 / (2 * step) / 30 + 30 * step ** 2
    zw = torch.randn(d, generator=gen, device="cuda")
    slope = (value(x, w + step * zw) - value(x, w - step * zw)) / (2 * step)
    assert abs(slope - (dw.double() * zw.double()).sum().item()) < 2e-5 / step + 30 * step ** 2


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_far_and_negative_positions(A, scaling):
    """Whole positions of any size turn by their angle without its whole turns."""
    plan = A.RotaryPlan(128, scaling=scaling, factor=32.0, original_length=4096, device="cuda")
    pos = torch.tensor([0, 1, -1, 4095, 131072, 1 << 20, -(1 << 20), 16777217], device="cuda")
    x = torch.randn(8, 2, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    y, none = A.rotary(x, None, pos, plan)
    assert none is None
    # the 64-bit reference itself: an angle of 2^24 has 2^24 * 2^-53 * 2, far below
    close(y, *turn(plan, x.double(), pos))
    back, _ = A.rotary_backward(y, None, pos, plan)
    assert torch.allclose(back.double(), x.double() * plan.amplitude ** 2, rtol=0, atol=32 * U * 6 * plan.amplitude ** 2)


def test_scaled_frequencies(A):
    base = A.RotaryPlan(64, device="cuda").inv_freq
    assert base == tuple(10000.0 ** (-2 * p / 64) for p in range(32))
    assert A.RotaryPlan(64, scaling="linear", factor=4.0, device="cuda").inv_freq == tuple(f / 4 for f in base)
    ntk = A.RotaryPlan(64, scaling="ntk", factor=4.0, device="cuda").inv_freq
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(base[-1] / 4, rel=1e-12)
    plan = A.RotaryPlan(64, scaling="yarn", factor=4.0, original_length=4096, device="cuda")
    for f, g in zip(base, plan.inv_freq):
        turns = 4096 * f / math.tau
        assert g == f if turns >= 32 else g == f / 4 if turns <= 1 else f / 4 < g < f
    assert plan.amplitude == pytest.approx(0.1 * math.log(4.0) + 1)
    own = A.RotaryPlan(4, inv_freq=[0.5, 7.0], amplitude=2.0, device="cuda")  # more than a turn a position
    x = torch.randn(3, 1, 4, device="cuda")
    close(A.rotary(x, None, torch.arange(3, device="cuda"), own)[0], *turn(own, x.double(), torch.arange(3, device="cuda")))


@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.int16])
def test_batches_share_positions(A, kind):
    gen = torch.Generator(device="cuda").manual_seed(5)
    plan = A.RotaryPlan(64, device="cuda")
    pos = torch.arange(100, 107, device="cuda", dtype=kind)
    for how in ("whole", "fused", "turned"):
        q, k = rows(gen, (3, 7, 4, 64), torch.bfloat16, how), rows(gen, (3, 7, 2, 64), torch.bfloat16, how)
        got = A.rotary(q, k, pos, plan)
        each = A.rotary(q, k, pos.expand(3, 7), plan)
        for g, e, x in zip(got, each, (q, k)):
            assert torch.equal(g, e) and g.shape == x.shape
            close(g, *turn(plan, x.double(), pos.expand(3, 7)))
    one = A.rotary(q, k, torch.tensor(5, device="cuda"), plan)[0]
    close(one, *turn(plan, q.double(), torch.full((3, 7), 5, device="cuda")))


def test_single_token_is_that_of_the_batch(A):
    """A token's result does not depend on the tokens beside it."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    plan = A.RotaryPlan(128, device="cuda")
    q, k = rows(gen, (513, 8, 128), torch.bfloat16, "fused"), rows(gen, (513, 2, 128), torch.bfloat16, "fused")
    w = torch.randn(128, generator=gen, device="cuda").bfloat16()
    pos = torch.arange(513, device="cuda") * 1000
    all_q, all_k = A.qk_norm_rotary(q, k, w, w, pos, plan)
    for i in (0, 1, 255, 512):
        one = A.qk_norm_rotary(q[i:i + 1], k[i:i + 1], w, w, pos[i:i + 1], plan)
        assert torch.equal(one[0][0], all_q[i]) and torch.equal(one[1][0], all_k[i])


def test_nothing_and_not_finite(A):
    plan = A.RotaryPlan(32, device="cuda")
    w = torch.ones(32, device="cuda")
    empty = torch.empty(0, 2, 32, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert A.rotary(empty, empty, none, plan)[0].shape == (0, 2, 32)
    out = A.qk_norm_rotary_backward(empty, empty, empty, empty, w, w, none, plan)
    assert (out[2] == 0).all() and (out[3] == 0).all()
    # zero rows stay zero, and a NaN stays in its own row
    x = torch.zeros(4, 2, 32, device="cuda")
    x[1, 1, 3] = float("nan")
    y, _ = A.qk_norm_rotary(x, None, w, None, torch.arange(4, device="cuda"), plan)
    bad = torch.isnan(y).any(-1)
    assert bad.nonzero().tolist() == [[1, 1]] and (y[~bad] == 0).all()


def test_stretches_of_many_rows(A):
    """More rows than a grid's first stretches, and a gradient whose CTAs take
    several: against the same rows in smaller calls."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    plan = A.RotaryPlan(64, device="cuda")
    n = 30011
    q, dq = (rows(gen, (n, 17, 64), torch.bfloat16, "whole") for _ in range(2))
    k, dk = (rows(gen, (n, 1, 64), torch.bfloat16, "whole") for _ in range(2))
    w = torch.randn(64, generator=gen, device="cuda")
    pos = torch.arange(n, device="cuda")
    got = A.qk_norm_rotary_backward(dq, dk, q, k, w, w, pos, plan)
    sums = [0.0, 0.0]
    for a in range(0, n, 10007):
        s = slice(a, a + 10007)
        part = A.qk_norm_rotary_backward(dq[s], dk[s], q[s], k[s], w, w, pos[s], plan)
        assert torch.equal(part[0], got[0][s]) and torch.equal(part[1], got[1][s])
        sums = [t + p.double() for t, p in zip(sums, part[2:])]
    for g, t, dy in zip(got[2:], sums, (dq, dk)):
        # |g x r| of a row is some 1 on average: n rows x 2^-24 each is far above what either order is off
        assert (g.double() - t).abs().max() < dy.shape[0] * dy.shape[1] * 4 * U
    again = A.qk_norm_rotary_backward(dq, dk, q, k, w, w, pos, plan)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("d, heads", [(128, 64), (33, 200)])
def test_more_features_than_32_bits_count(A, d, heads):
    """Tokens on both sides of feature 2^31: as alone."""
    gen = torch.Generator(device="cuda").manual_seed(13)
    plan = A.RotaryPlan(32, device="cuda")
    n = 2 ** 31 // (heads * d) + 37
    q, dq = (torch.empty(n, heads, d, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2))
    w = torch.randn(d, generator=gen, device="cuda")
    pos = torch.arange(n, device="cuda")
    s = slice(n - 80, n)
    assert torch.equal(A.rotary(q, None, pos, plan)[0][s], A.rotary(q[s], None, pos[s], plan)[0])
    assert torch.equal(A.qk_norm_rotary(q, None, w, None, pos, plan)[0][s], A.qk_norm_rotary(q[s], None, w, None, pos[s], plan)[0])
    assert torch.equal(A.qk_norm_rotary_backward(dq, None, q, None, w, None, pos, plan)[0][s],
                       A.qk_norm_rotary_backward(dq[s], None, q[s], None, w, None, pos[s], plan)[0])


@pytest.mark.parametrize("heads", [511, 512, 513, 32768, 32769, 40000])
def test_many_heads(A, heads):
    """Heads in the thousands, whose rows' tokens come by a product or a comparison."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    for d, r in ((16, 16), (6, 4)):
        plan = A.RotaryPlan(r, device="cuda")
        pos = torch.tensor([3, 70000, 12], device="cuda")
        q, dq = (torch.randn(3, heads, d, generator=gen, device="cuda") for _ in range(2))
        w = 1 + 0.1 * torch.randn(d, generator=gen, device="cuda")
        close(A.rotary(q, q[:, :5], pos, plan)[0], *turn(plan, q.double(), pos), (heads, d))
        dx, _, dw, _ = A.qk_norm_rotary_backward(dq, None, q, None, w, None, pos, plan)
        g, _ = turn(plan, dq.double(), pos, -1.0)
        x = q.double()
        rr = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        want = rr * w * g - x * rr ** 3 * (w * g * x).mean(-1, keepdim=True)
        # of sizes of 1 to 10 in fp32: far below 1e-4
        assert (dx.double() - want).abs().max() < 1e-4 and (dw.double() - (g * x * rr).sum((0, 1))).abs().max() < 3 * heads * 1e-6


def test_captured(A):
    gen = torch.Generator(device="cuda").manual_seed(8)
    plan = A.RotaryPlan(64, device="cuda")
    q, k = rows(gen, (9, 4, 64), torch.float16, "fused"), rows(gen, (9, 2, 64), torch.float16, "fused")
    w = torch.randn(64, generator=gen, device="cuda").half()
    pos = torch.arange(9, device="cuda")

    def call():
        y = A.qk_norm_rotary(q, k, w, w, pos, plan)
        return (*y, *A.qk_norm_rotary_backward(*y, q, k, w, w, pos, plan), *A.rotary(q, k, pos, plan))

    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    pos += 1000
    q.mul_(0.5)
    graph.replay()
    for a, b in zip(got, call()):
        assert torch.equal(a, b)


def test_refusals(A):
    plan = A.RotaryPlan(32, device="cuda")
    q, k, pos, w = (torch.zeros(4, 2, 32, device="cuda"), torch.zeros(4, 1, 32, device="cuda"),
                    torch.arange(4, device="cuda"), torch.ones(32, device="cuda"))
    for bad in ((q.int(), k, pos, plan), (q, k.half(), pos, plan), (q, k[:3], pos, plan), (q[..., :16], k[..., :16], pos, plan),
                (q, k, pos[:3], plan), (q, k, pos.float(), plan), (q, k, pos.cpu(), plan), (q, k.cpu(), pos, plan),
                (q, k, pos > 1, plan), (q, k, pos, A.RotaryPlan(32)), (q, k, pos, None), (q[:, :0], k, pos, plan),
                (torch.zeros(4, 1, 1025, device="cuda"), None, pos, plan), (q, k, pos[:, None], plan)):
        with pytest.raises(ValueError):
            A.rotary(*bad)
    for wq, wk in ((w[:16], w), (w, None), (w, w.half()), (w.int(), w.int()), (w, w.cpu()), (w, w[None])):
        with pytest.raises(ValueError):
            A.qk_norm_rotary(q, k, wq, wk, pos, plan)
    for dq, dk in ((q[:3], k), (q.half(), k), (q, None)):
        with pytest.raises(ValueError):
            A.qk_norm_rotary_backward(dq, dk, q, k, w, w, pos, plan)
