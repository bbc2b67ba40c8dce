"""The checkpointed RMS norm, its restoring and gradient, and the weight gradient
from the checkpoint, against the definitions in 64 bits.

Codes and scales are compared bit for bit with the formula in 32 bits (each of
its operations rounds once).  Other tolerances (u = 2^-8 bf16, 2^-11 f16, 2^-24
f32, half an ulp relative): a sum of d squares or products in fp32 is within
(d / 8 + 16) 2^-24 of its terms' magnitudes (at least eight partial sums a row,
then a tree); the norm's factor takes half of that and four roundings more;
outputs are rounded once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}
E = 2.0 ** -24
EPS = 1e-6
ALL = [torch.bfloat16, torch.float16, torch.float32]


def acts(rows, d, dt, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, d, generator=gen, device="cuda")
    x[:, torch.randint(0, d, (max(1, d // 100),), generator=gen, device="cuda")] *= 30.0
    return x.to(dt), (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")), gen


def formula_codes(x):
    """Codes and scales from the 32-bit formula, in numpy."""
    x = x.float().cpu().numpy()
    rows, d = x.shape
    nb = -(-d // 128)
    p = np.zeros((rows, nb * 128), np.float32)
    p[:, :d] = x
    p = p.reshape(rows, nb, 128)
    amax = np.abs(p).max(2)
    scale = np.where(amax < np.float32(2.0 ** -119), np.float32(1), amax / np.float32(127)).astype(np.float32)
    v = p * (np.float32(1) / scale)[:, :, None]
    t = np.trunc(v)
    q = np.clip(t + np.sign(v) * (np.abs(v - t) >= 0.5), -127, 127).astype(np.int8)
    return q.reshape(rows, -1)[:, :d], scale


def close(got, want, bound):
    assert got.isfinite().all()
    off = (got.double() - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def norm64(x, gain):
    return x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * gain


def norm_bound(y, d, dt):
    return y.abs() * (1.1 * U[dt] + (d / 16 + 16) * E) + TINY[dt]


def values64(ck):
    d = ck.codes.shape[-1]
    return ck.codes.double() * ck.scales.double().repeat_interleave(128, -1)[..., :d]


SHAPES = [(1, 1), (1, 4096), (2, 127), (3, 128), (5, 129), (33, 1000), (64, 2048), (7, 5120), (300, 257), (20, 8192), (4, 12300),
          (3, 20000), (2, 40001)]


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,d", SHAPES)
def test_store_and_restore(dt, rows, d):
    import aethelstream_b200 as A
    x, gain, _ = acts(rows, d, dt, rows + d)
    for gdt in (dt, torch.float32):
        g = gain.to(gdt)
        y, ck = A.rms_norm_checkpoint(x, g, eps=EPS)
        close(y, norm64(x.double(), g.double()), norm_bound(norm64(x.double(), g.double()), d, dt))
    q, s = formula_codes(x)
    assert np.array_equal(ck.codes.cpu().numpy(), q) and np.array_equal(ck.scales.cpu().numpy(), s)
    v = values64(ck)
    assert torch.equal(A.checkpoint_decode(ck), (ck.codes.float() * ck.scales.repeat_interleave(128, 1)[:, :d]).to(dt))
    want = norm64(v, g.double())
    close(A.checkpoint_decode(ck, norm_weight=g, eps=EPS), want, norm_bound(want, d, dt) * 1.05)
    # what 8 bits cost: half a step of the block
    step = ck.scales.repeat_interleave(128, 1)[:, :d].double()
    assert ((v - x.double()).abs() <= 0.5 * step * (1 + 1e-5)).all()


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,d", [(1, 64), (3, 129), (130, 1000), (9, 8192), (2, 20000)])
def test_store_with_residual(dt, rows, d):
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, dt, 5)
    res = torch.randn(rows, d, generator=gen, device="cuda").to(dt)
    g = gain.to(dt)
    y, ck, total = A.rms_norm_checkpoint(x, g, eps=EPS, residual=res)
    assert torch.equal(total, (x.float() + res.float()).to(dt))
    y2, ck2 = A.rms_norm_checkpoint(total, g, eps=EPS)
    assert torch.equal(y, y2) and torch.equal(ck.codes, ck2.codes) and torch.equal(ck.scales, ck2.scales)


def back64(x, dy, gain, res):
    d = x.shape[1]
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    dyw = dy * gain
    dx = r * dyw - x * r ** 3 * (dyw * x).mean(1, keepdim=True)
    e = (d / 8 + 24) * E
    bound = e * (r * dyw.abs() + x.abs() * r ** 3 * (dyw * x).abs().mean(1, keepdim=True) * 2)
    if res is not None:
        dx = dx + res
        bound = bound + 2 * E * (res.abs() + dx.abs())
    return dx, bound, (dy * x * r).sum(0), (dy * x * r).abs().sum(0) * ((d / 16 + 16) + x.shape[0]) * E


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,d", SHAPES + [(1000, 384), (2500, 64)])
@pytest.mark.parametrize("with_res", [False, True])
def test_backward(dt, rows, d, with_res):
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, dt, rows * 3 + d)
    _, ck = A.rms_norm_checkpoint(x, gain.to(dt), eps=EPS)
    dy = torch.randn(rows, d, generator=gen, device="cuda").to(dt)
    res = torch.randn(rows, d, generator=gen, device="cuda").to(dt) if with_res else None
    for g in (gain.to(dt), gain):
        dx, dw = A.rms_norm_checkpoint_backward(dy, ck, g, eps=EPS, d_residual=res)
        want, bound, want_w, bound_w = back64(values64(ck), dy.double(), g.double(), None if res is None else res.double())
        close(dx, want, 1.1 * (bound + U[dt] * want.abs()) + TINY[dt])
        close(dw, want_w, bound_w + 1e-37)
    again = A.rms_norm_checkpoint_backward(dy, ck, gain, eps=EPS, d_residual=res)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_backward_against_differences():
    import aethelstream_b200 as A
    x, gain, gen = acts(40, 200, torch.float32, 1)
    _, ck = A.rms_norm_checkpoint(x, gain, eps=EPS)
    dy = torch.randn(40, 200, generator=gen, device="cuda")
    dx, dw = A.rms_norm_checkpoint_backward(dy, ck, gain, eps=EPS)
    v, g = values64(ck), gain.double()
    _, b_x, _, b_w = back64(v, dy.double(), g, None)
    f = lambda a, b: (norm64(a, b) * dy.double()).sum()  # noqa: E731
    h = 1e-5
    for got, bound, e in ((dx, b_x, torch.randn(40, 200, generator=gen, device="cuda").double()),
                          (dw, b_w, torch.randn(200, generator=gen, device="cuda").double())):
        diff = (f(v + h * e, g) - f(v - h * e, g)) if got is dx else (f(v, g + h * e) - f(v, g - h * e))
        along = (got.double() * e).sum()
        assert abs(along - diff / (2 * h)) <= ((bound + 2 * E * got.double().abs()) * e.abs()).sum() + 1e-5 * along.abs() * h + 1e-6


def test_zero_tiny_and_non_finite_blocks():
    import aethelstream_b200 as A
    x = torch.randn(6, 300, device="cuda")
    x[0] = 0.0
    x[1, :128] = 0.0
    x[2, 128:256] = 1e-38
    x[3, 5] = float("nan")
    x[4, 200] = float("inf")
    x[5, 299] = float("-inf")
    y, ck = A.rms_norm_checkpoint(x, torch.ones(300, device="cuda"))
    s, r = ck.scales, A.checkpoint_decode(ck)
    assert (s[0] == 1).all() and (r[0] == 0).all() and (y[0] == 0).all()
    assert s[1, 0] == 1 and (r[1, :128] == 0).all() and s[2, 1] == 1 and (r[2, 128:256] == 0).all()
    assert s[3].isnan().tolist() == [True, False, False] and r[3, :128].isnan().all() and r[3, 128:].isfinite().all()
    assert s[4].isnan().tolist() == [False, True, False] and r[4, 128:256].isnan().all()
    assert s[5].isnan().tolist() == [False, False, True] and r[5, 256:].isnan().all()
    assert y[3].isnan().all() and y[:3].isfinite().all()


@pytest.mark.parametrize("dt", ALL)
def test_strides_and_odd_addresses(dt):
    """Row strides, column slices and addresses that vectors cannot take."""
    import aethelstream_b200 as A
    x, gain, gen = acts(24, 513, dt, 2)
    big = torch.zeros(48, 1031, dtype=dt, device="cuda")
    big[::2, 5:518] = x
    xs = big[::2, 5:518]
    pad = torch.zeros(514, device="cuda").to(dt)
    pad[1:] = gain.to(dt)
    g = pad[1:]
    for a, b in zip(A.rms_norm_checkpoint(xs.view(4, 6, 513), g), A.rms_norm_checkpoint(x, g.clone())):
        if isinstance(a, A.ActivationCheckpoint):
            ck = b
            assert torch.equal(a.codes.view(24, 513), b.codes) and torch.equal(a.scales.view(24, -1), b.scales)
        else:
            assert a.shape == (4, 6, 513) and torch.equal(a.view(24, 513), b)
    dy = torch.randn(24, 513, generator=gen, device="cuda").to(dt)
    bigd = torch.zeros(24, 700, dtype=dt, device="cuda")
    bigd[:, 3:516] = dy
    a = A.rms_norm_checkpoint_backward(bigd[:, 3:516], ck, g, d_residual=xs)
    b = A.rms_norm_checkpoint_backward(dy, ck, g.clone(), d_residual=x)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    buf = torch.zeros(24 * 513 + 3, dtype=torch.int8, device="cuda")
    buf[3:] = ck.codes.view(-1)
    odd = A.ActivationCheckpoint(buf[3:].view(24, 513), ck.scales, dt)
    assert torch.equal(A.checkpoint_decode(odd), A.checkpoint_decode(ck))
    c = A.rms_norm_checkpoint_backward(dy, odd, g, d_residual=x)
    assert torch.equal(c[0], b[0]) and torch.equal(c[1], b[1])


def test_no_rows():
    import aethelstream_b200 as A
    x = torch.empty(0, 64, device="cuda")
    g = torch.ones(64, device="cuda")
    y, ck = A.rms_norm_checkpoint(x, g)
    assert y.shape == (0, 64) and ck.scales.shape == (0, 1) and A.checkpoint_decode(ck).shape == (0, 64)
    dx, dw = A.rms_norm_checkpoint_backward(x, ck, g)
    assert dx.shape == (0, 64) and (dw == 0).all()
    ck16 = A.ActivationCheckpoint(ck.codes, ck.scales, torch.bfloat16)
    dW = A.checkpoint_weight_grad(torch.empty(0, 24, dtype=torch.bfloat16, device="cuda"), ck16)
    assert dW.shape == (24, 64) and (dW == 0).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,m,d", [(1, 8, 64), (1, 300, 520), (7, 64, 129), (63, 33, 200), (64, 256, 256), (65, 257, 1000),
                                      (300, 1000, 264), (1001, 520, 96), (2050, 72, 2056), (4096, 256, 256)])
@pytest.mark.parametrize("norm", [False, True])
def test_weight_grad(dt, rows, m, d, norm):
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, dt, rows + m + d)
    g = gain.to(dt)
    _, ck = A.rms_norm_checkpoint(x, g, eps=EPS)
    dy = torch.randn(rows, m, generator=gen, device="cuda").to(dt)
    dw = A.checkpoint_weight_grad(dy, ck, norm_weight=g if norm else None, eps=EPS)
    v = values64(ck)
    e = 1.1 * U[dt] + 2.0 ** -22
    if norm:
        v, e = norm64(v, g.double()), e + (d / 16 + 16) * E
    want = dy.double().T @ v
    mag = dy.double().abs().T @ v.abs()
    close(dw, want, (e + 2 * rows * E) * mag + 1.1 * U[dt] * want.abs() + TINY[dt] * (1 + dy.double().abs().sum(0)[:, None]))
    assert dw.dtype == dt and dw.shape == (m, d)
    assert torch.equal(dw, A.checkpoint_weight_grad(dy, ck, norm_weight=g if norm else None, eps=EPS))
    wide = torch.zeros(rows, m + 11, dtype=dt, device="cuda")
    wide[:, 5:m + 5] = dy
    assert torch.equal(dw, A.checkpoint_weight_grad(wide[:, 5:m + 5], ck, norm_weight=g if norm else None, eps=EPS))


def test_graph_and_stream():
    import aethelstream_b200 as A
    x, gain, gen = acts(500, 1024, torch.bfloat16, 3)
    g = gain.bfloat16()
    dy = torch.randn(500, 1024, generator=gen, device="cuda").bfloat16()

    def path():
        y, ck, s = A.rms_norm_checkpoint(x, g, residual=dy)
        dx, dg = A.rms_norm_checkpoint_backward(dy, ck, g, d_residual=s)
        return y, s, ck.codes, A.checkpoint_decode(ck, g), dx, dg, A.checkpoint_weight_grad(dy, ck, g)

    first = path()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = path()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = path()
    for t in third:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_offsets_beyond_32_bits():
    """2.2e9 activations; the last rows equal the same rows alone."""
    import aethelstream_b200 as A
    rows, d = 270000, 8192
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda")
    x[-40:] = torch.randn(40, d, device="cuda").bfloat16()
    g = torch.ones(d, dtype=torch.bfloat16, device="cuda")
    y, ck = A.rms_norm_checkpoint(x, g)
    y1, ck1 = A.rms_norm_checkpoint(x[-40:], g)
    assert torch.equal(y[-40:], y1) and torch.equal(ck.codes[-40:], ck1.codes) and torch.equal(ck.scales[-40:], ck1.scales)
    dx, dw = A.rms_norm_checkpoint_backward(x, ck, g)
    dx1, dw1 = A.rms_norm_checkpoint_backward(x[-40:], ck1, g)
    assert torch.equal(dx[-40:], dx1)
    assert ((dw - dw1).abs() <= 1e-4 * (1 + dw1.abs())).all()
    assert torch.equal(A.checkpoint_decode(ck)[-40:], A.checkpoint_decode(ck1))


@pytest.mark.parametrize("rows,d", [(9, 64), (333, 64), (701, 200), (5, 9000)])
def test_backward_without_eps(rows, d):
    """eps = 0: rows that a CTA holds past the last one add nothing to d_weight."""
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, torch.float32, 8)
    _, ck = A.rms_norm_checkpoint(x, gain, eps=0.0)
    dy = torch.randn(rows, d, generator=gen, device="cuda")
    dx, dw = A.rms_norm_checkpoint_backward(dy, ck, gain, eps=0.0)
    v = values64(ck)
    want = (dy.double() * v / torch.sqrt((v * v).mean(1, keepdim=True)))
    close(dw, want.sum(0), want.abs().sum(0) * (d / 16 + 16 + rows) * E + 1e-37)
    assert dx.isfinite().all()


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,d", [(333, 8208), (700, 12288), (301, 16384), (1200, 1008), (900, 5120)])
@pytest.mark.parametrize("with_res", [False, True])
def test_backward_of_many_rows(dt, rows, d, with_res):
    """Against the formula, and bit for bit what the first rows give by themselves."""
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, dt, rows + d)
    _, ck = A.rms_norm_checkpoint(x, gain.to(dt), eps=EPS)
    dy = torch.randn(rows, d, generator=gen, device="cuda").to(dt)
    res = torch.randn(rows, d, generator=gen, device="cuda").to(dt) if with_res else None
    dx, dw = A.rms_norm_checkpoint_backward(dy, ck, gain, eps=EPS, d_residual=res)
    want, bound, want_w, bound_w = back64(values64(ck), dy.double(), gain.double(), None if res is None else res.double())
    close(dx, want, 1.1 * (bound + U[dt] * want.abs()) + TINY[dt])
    close(dw, want_w, bound_w + 1e-37)
    few = A.rms_norm_checkpoint(x[:9], gain.to(dt), eps=EPS)[1]
    assert torch.equal(A.rms_norm_checkpoint_backward(dy[:9], few, gain, eps=EPS,
                                                      d_residual=None if res is None else res[:9])[0], dx[:9])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,m,d", [(8170, 216, 952), (5000, 64, 64), (8000, 33, 1001), (8191, 1032, 1040), (8192, 4608, 4360)])
def test_weight_grad_split_along_the_tokens(dt, rows, m, d):
    """Tiles that leave CTA pairs idle, alone and after whole waves."""
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, dt, rows + m + d)
    _, ck = A.rms_norm_checkpoint(x, gain.to(dt), eps=EPS)
    dy = torch.randn(rows, m, generator=gen, device="cuda").to(dt)
    dw = A.checkpoint_weight_grad(dy, ck)
    v = values64(ck)
    want = dy.double().T @ v
    mag = dy.double().abs().T @ v.abs()
    close(dw, want, (1.1 * U[dt] + 2.0 ** -22 + 2 * rows * E) * mag + 1.1 * U[dt] * want.abs()
          + TINY[dt] * (1 + dy.double().abs().sum(0)[:, None]))
    assert torch.equal(dw, A.checkpoint_weight_grad(dy, ck))


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,d", [(5, 1), (40, 7), (3, 8), (9, 255), (9, 257), (33, 263), (700, 513), (400, 2276), (350, 8191), (4, 9001)])
def test_rows_off_alignment(dt, rows, d):
    """Every width and address gives bit for bit what aligned rows give."""
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, dt, rows + d)
    g = gain.to(dt)
    dy = torch.randn(rows, d, generator=gen, device="cuda").to(dt)
    p = -(-d // 16) * 16  # the same rows with zeros up to a multiple of 16: the same blocks and codes

    def padded(t):
        o = torch.zeros(t.shape[:-1] + (p,), dtype=t.dtype, device="cuda")
        o[..., :d] = t
        return o

    ck, ck_p = A.rms_norm_checkpoint(x, g, residual=dy)[1], A.rms_norm_checkpoint(padded(x), padded(g), residual=padded(dy))[1]
    assert torch.equal(ck.codes, ck_p.codes[:, :d]) and torch.equal(ck.scales, ck_p.scales)
    plain = A.checkpoint_decode(ck)
    assert torch.equal(plain, A.checkpoint_decode(ck_p)[:, :d])
    total = A.rms_norm_checkpoint(x, g, residual=dy)[2]
    assert torch.equal(total, (x.float() + dy.float()).to(dt))
    first = A.rms_norm_checkpoint(x, g, eps=EPS), A.checkpoint_decode(ck, g, eps=EPS)
    dx, dw = A.rms_norm_checkpoint_backward(dy, ck, g, eps=EPS, d_residual=x)
    for shift in range(1, 9):
        wide = torch.zeros(rows, d + 19, dtype=dt, device="cuda")
        wide[:, shift:shift + d] = x
        dwide = torch.zeros(rows, d + 13, dtype=dt, device="cuda")
        dwide[:, shift:shift + d] = dy
        xs, ds = wide[:, shift:shift + d], dwide[:, shift:shift + d]
        y, c = A.rms_norm_checkpoint(xs, g, eps=EPS)
        assert torch.equal(y, first[0][0]) and torch.equal(c.codes, first[0][1].codes) and torch.equal(c.scales, first[0][1].scales)
        dxs, dws = A.rms_norm_checkpoint_backward(ds, ck, g, eps=EPS, d_residual=xs)
        assert torch.equal(dxs, dx) and torch.equal(dws, dw)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,d", [(9, 1000), (500, 257), (700, 1008), (400, 12288), (3, 20000)])
@pytest.mark.parametrize("size,eps", [(1e15, EPS), (1e-18, 0.0)])
def test_backward_of_large_and_small_activations(dt, rows, d, size, eps):
    """Activations whose squares fp32 holds, though not the factor's third power."""
    import aethelstream_b200 as A
    x, gain, gen = acts(rows, d, torch.float32, rows + d)
    x = (x * size).to(dt)
    _, ck = A.rms_norm_checkpoint(x, gain.to(dt), eps=eps)
    dy = torch.randn(rows, d, generator=gen, device="cuda").to(dt)
    dx, dw = A.rms_norm_checkpoint_backward(dy, ck, gain, eps=eps)
    v, dyw = values64(ck), dy.double() * gain.double()
    r = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    want = r * dyw - v * r ** 3 * (dyw * v).mean(1, keepdim=True)
    bound = (d / 8 + 24) * E * (r * dyw.abs() + v.abs() * r ** 3 * (dyw * v).abs().mean(1, keepdim=True) * 2)
    close(dx, want, 1.1 * (bound + U[dt] * want.abs()) + TINY[dt])
    t = dy.double() * v * r
    close(dw, t.sum(0), t.abs().sum(0) * ((d / 16 + 16) + rows) * E + 1e-37)
