"""The head's cross entropy and its gradient against the definition in 64 bits.

Tolerances (u = 2^-8 for bf16, 2^-11 for f16, half an ulp relative):
  logits: fp32 sums of exact products, within 2 d 2^-24 * sum_i |h_i w_i| of the
    exact one (twice the bound of a rounded sum: the tensor cores' own order and
    rounding are not specified);
  loss and lse: the logits' bound twice, and 2^-18 (1 + |lse|) for the
    exponentials and the logarithm;
  G: relative u (rounded once) and the error of its exponent, i.e. twice the
    logits' bound, and the exponential's; times |W| or |H| and summed;
  outputs: rounded once more, u |x|, and f16's spacing near zero."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
IGNORE = -100


def make(n, d, v, dt, seed, masked=0.0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = (scale * torch.randn(n, d, generator=gen, device="cuda")).to(dt)
    w = (torch.randn(v, d, generator=gen, device="cuda") * (2.0 / d ** 0.5)).to(dt)
    lab = torch.randint(0, v, (n,), generator=gen, device="cuda")
    lab[torch.rand(n, generator=gen, device="cuda") < masked] = IGNORE
    return h, w, lab


def reference(h, w, lab, grad=None, scale=1.0):
    """Losses, lse, mean, G, dH, dW in 64 bits, and the bounds."""
    dt = h.dtype
    n, d = h.shape
    keep = lab != IGNORE
    hd = torch.where(keep[:, None], h, torch.zeros_like(h)).double()
    wd = w.double()
    s = hd @ wd.T
    lse = torch.logsumexp(s, 1)
    at = torch.where(keep, lab, 0)[:, None]
    losses = torch.where(keep, lse - s.gather(1, at)[:, 0], 0.0)
    count = max(int(keep.sum()), 1)
    g_t = torch.full((n,), scale / count, dtype=torch.float64, device="cuda") if grad is None else scale * grad.double()
    g_t = torch.where(keep, g_t, 0.0)
    G = torch.softmax(s, 1)
    G.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float64))
    G *= g_t[:, None]
    e_s = (hd.abs() @ wd.abs().T).amax(1) * (2 * d * 2.0 ** -24)
    e_loss = 2 * e_s + 2.0 ** -18 * (1 + lse.abs())
    # error of an entry of G: relative, of p = G + onehot g_t
    p = G.clone()
    p.scatter_add_(1, at, g_t[:, None])
    e_g = G.abs() * (U[dt] + 2.0 ** -20) + p.abs() * (2 * e_s + 2.0 ** -18)[:, None]
    if dt is torch.float16:
        e_g += 2.0 ** -40 * g_t.abs().max()
    dh, dw = G @ wd, G.T @ hd
    tiny = 2.0 ** -24 if dt is torch.float16 else 1e-38
    acc = 2 * 2.0 ** -24
    b_h = 1.1 * (e_g @ wd.abs()) + acc * w.shape[0] * (G.abs() @ wd.abs()) + 1.1 * U[dt] * dh.abs() + tiny
    b_w = 1.1 * (e_g.T @ hd.abs()) + acc * n * (G.abs().T @ hd.abs()) + 1.1 * U[dt] * dw.abs() + tiny
    return dict(losses=losses, lse=lse, loss=losses.sum() / count, dh=dh, dw=dw, e_loss=e_loss, b_h=b_h, b_w=b_w, keep=keep)


def close(got, want, bound):
    off = (got.double() - want).abs()
    assert got.isfinite().all()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def check(h, w, lab, grad=None, scale=1.0, ref_inputs=None):
    import aethelstream_b200 as A
    ce = A.cut_cross_entropy(h, w, lab, ignore_index=IGNORE)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=grad, scale=scale, ignore_index=IGNORE)
    r = reference(*(ref_inputs or (h, w, lab)), grad=grad, scale=scale)
    close(ce.losses, r["losses"], r["e_loss"])
    close(ce.lse, torch.where(r["keep"], r["lse"], 0.0), r["e_loss"])
    close(ce.loss, r["loss"], r["e_loss"].max())
    close(dh, r["dh"], r["b_h"])
    close(dw, r["dw"], r["b_w"])
    assert dh.dtype == h.dtype and dw.dtype == w.dtype
    return ce, dh, dw


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d,v", [(1, 64, 1000), (1, 8, 7), (2, 40, 255), (3, 136, 257), (63, 512, 4099), (64, 64, 256),
                                   (65, 200, 513), (130, 96, 1), (255, 64, 300), (257, 1032, 700), (520, 72, 2049),
                                   (1000, 256, 77)])
def test_sizes(dt, n, d, v):
    check(*make(n, d, v, dt, seed=n + d + v))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d,v", [(5, 33, 130), (70, 1, 64), (40, 129, 1001)])
def test_widths_that_tma_cannot_read_in_place(dt, n, d, v):
    check(*make(n, d, v, dt, seed=n))


@pytest.mark.parametrize("masked", [0.3, 0.9, 1.0])
@pytest.mark.parametrize("n", [1, 40, 300, 700])
def test_masked_tokens_take_no_part(n, masked):
    """NaN and infinities in masked rows reach nothing; masked rows get zeros."""
    h, w, lab = make(n, 128, 600, torch.bfloat16, seed=n, masked=masked)
    bad = h.clone()
    out = lab == IGNORE
    bad[out] = float("nan")
    bad[out & (torch.arange(n, device="cuda") % 2 == 0)] = float("inf")
    ce, dh, dw = check(bad, w, lab, ref_inputs=(h, w, lab))
    assert (ce.losses[out] == 0).all() and (dh[out] == 0).all()
    if out.all():
        assert ce.loss.item() == 0 and (dw == 0).all()


def test_pieces_of_the_vocabulary():
    """More logits than one piece of G holds: 4200 tokens x 40001 entries."""
    check(*make(4200, 64, 40001, torch.bfloat16, seed=2, masked=0.02))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_token_weights_and_scale(dt):
    h, w, lab = make(200, 128, 1000, dt, seed=9, masked=0.1)
    gen = torch.Generator(device="cuda").manual_seed(1)
    grad = torch.randn(200, generator=gen, device="cuda") * torch.logspace(-3, 0, 200, device="cuda")
    grad[7] = 0.0
    check(h, w, lab, grad=grad, scale=8.0)
    check(h, w, lab, scale=-3.0)


def test_all_token_weights_zero():
    import aethelstream_b200 as A
    h, w, lab = make(20, 64, 100, torch.bfloat16, seed=3)
    ce = A.cut_cross_entropy(h, w, lab)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=torch.zeros(20, device="cuda"))
    assert (dh == 0).all() and (dw == 0).all()


def test_large_logits_and_lowest_entries():
    """Logits of hundreds, and vocabulary entries pushed to the type's lowest
    value by a constant feature (padding of the vocabulary): whole tiles of it."""
    h, w, lab = make(90, 64, 1500, torch.bfloat16, seed=4, scale=60.0)
    check(h, w, lab)
    h, w, lab = make(90, 64, 1500, torch.bfloat16, seed=5)
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    w[700:, 0] = torch.finfo(torch.bfloat16).min
    lab = lab % 700
    import aethelstream_b200 as A
    ce = A.cut_cross_entropy(h, w, lab)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce)
    r = reference(h, w[:700], lab)
    close(ce.losses, r["losses"], r["e_loss"])
    close(dh[:, 1:], r["dh"][:, 1:], r["b_h"][:, 1:])
    close(dw[:700], r["dw"], r["b_w"])
    assert (dw[700:] == 0).all() and dh[:, 0].isfinite().all()


def test_a_live_token_that_is_not_finite():
    """Its own loss is NaN; the other tokens' losses and gradients stand."""
    import aethelstream_b200 as A
    h, w, lab = make(70, 64, 500, torch.bfloat16, seed=6)
    good = A.cut_cross_entropy(h, w, lab)
    h2 = h.clone()
    h2[33, 5] = float("nan")
    ce = A.cut_cross_entropy(h2, w, lab)
    others = torch.arange(70, device="cuda") != 33
    assert ce.losses[33].isnan() and ce.loss.isnan() and torch.equal(ce.losses[others], good.losses[others])
    dh, _ = A.cut_cross_entropy_backward(h2, w, lab, ce)
    assert dh[33].isnan().all() and dh[others].isfinite().all()


def test_label_outside_the_vocabulary():
    import aethelstream_b200 as A
    from aethelstream_b200 import _lib as L
    L.device_error_bits(0)
    h, w, lab = make(30, 64, 100, torch.bfloat16, seed=7)
    good = A.cut_cross_entropy(h, w, lab)
    lab2 = lab.clone()
    lab2[3], lab2[4] = 100, -7
    ce = A.cut_cross_entropy(h, w, lab2)
    assert ce.losses[3:5].isnan().all() and ce.loss.isnan() and torch.equal(ce.losses[5:], good.losses[5:])
    dh, dw = A.cut_cross_entropy_backward(h, w, lab2, ce)
    assert (dh[3:5] == 0).all() and dh.isfinite().all() and dw.isfinite().all()
    assert L.device_error_bits(0) == L.DEVERR_BAD_ARG and L.device_error_bits(0) == 0


def test_strides_shapes_and_label_types():
    """Batched shapes, a column slice, a row stride, an odd address, int32 labels."""
    import aethelstream_b200 as A
    h, w, lab = make(24, 64, 300, torch.bfloat16, seed=8, masked=0.2)
    ce, dh, dw = check(h, w, lab)
    wide = torch.randn(48, 131, device="cuda").bfloat16()
    wide[::2, 67:] = h
    ww = torch.randn(300, 70, device="cuda").bfloat16()
    ww[:, 3:67] = w
    hs, ws = wide[::2, 67:], ww[:, 3:67]
    ce2 = A.cut_cross_entropy(hs.unflatten(0, (4, 6)), ws, lab.int().view(4, 6))
    dh2, dw2 = A.cut_cross_entropy_backward(hs.unflatten(0, (4, 6)), ws, lab.int().view(4, 6), ce2)
    assert ce2.losses.shape == (4, 6) and dh2.shape == (4, 6, 64)
    assert torch.equal(ce2.losses.view(-1), ce.losses) and torch.equal(dh2.view(24, 64), dh) and torch.equal(dw2, dw)
    one = h[:1].T.contiguous().T  # a single row whose stride says nothing
    assert torch.equal(A.cut_cross_entropy(one, w, lab[:1]).lse, A.cut_cross_entropy(h[:1], w, lab[:1]).lse)


def test_no_tokens():
    import aethelstream_b200 as A
    h, w, lab = make(1, 64, 300, torch.bfloat16, seed=8)
    ce = A.cut_cross_entropy(h[:0], w, lab[:0])
    dh, dw = A.cut_cross_entropy_backward(h[:0], w, lab[:0], ce)
    assert ce.loss.item() == 0 and ce.losses.shape == (0,) and dh.shape == (0, 64) and (dw == 0).all()


def test_only_one_gradient():
    import aethelstream_b200 as A
    h, w, lab = make(150, 96, 700, torch.float16, seed=10)
    ce = A.cut_cross_entropy(h, w, lab)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce)
    a, none = A.cut_cross_entropy_backward(h, w, lab, ce, need_weight=False)
    assert none is None and torch.equal(a, dh)
    none, b = A.cut_cross_entropy_backward(h, w, lab, ce, need_hidden=False)
    assert none is None and torch.equal(b, dw)


def test_same_bits_again_on_another_stream_and_in_a_graph():
    import aethelstream_b200 as A
    h, w, lab = make(400, 256, 3000, torch.bfloat16, seed=11, masked=0.3)

    def step():
        ce = A.cut_cross_entropy(h, w, lab)
        return (ce.loss, ce.losses, *A.cut_cross_entropy_backward(h, w, lab, ce))

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    for t in third:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gradient_against_differences(dt):
    """Central differences of the definition in 64 bits along random directions."""
    import aethelstream_b200 as A
    h, w, lab = make(60, 64, 200, dt, seed=12, masked=0.2)
    ce = A.cut_cross_entropy(h, w, lab)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce)
    r = reference(h, w, lab)
    keep = lab != IGNORE

    def loss(hd, wd):
        return torch.nn.functional.cross_entropy(hd @ wd.T, lab, ignore_index=IGNORE)

    gen = torch.Generator(device="cuda").manual_seed(3)
    for x, got, bound in ((h, dh, r["b_h"]), (w, dw, r["b_w"])):
        e = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
        if x is h:
            e[~keep] = 0.0
        step = 1e-5
        hd, wd = h.double(), w.double()
        up = loss(hd + step * e, wd) if x is h else loss(hd, wd + step * e)
        dn = loss(hd - step * e, wd) if x is h else loss(hd, wd - step * e)
        diff = ((up - dn) / (2 * step)).item()
        along = (got.double() * e).sum().item()
        assert abs(along - diff) <= (bound * e.abs()).sum().item() + 1e-8


def test_offsets_beyond_32_bits():
    """A weight of 2.2e9 elements: the last entries' logits and gradients."""
    import aethelstream_b200 as A
    n, d, v = 3, 8192, 270001
    gen = torch.Generator(device="cuda").manual_seed(13)
    h = torch.randn(n, d, generator=gen, device="cuda").bfloat16()
    w = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    w[-500:] = (torch.randn(500, d, generator=gen, device="cuda") * 0.05).bfloat16()
    lab = torch.tensor([v - 1, v - 400, 5], device="cuda")
    ce = A.cut_cross_entropy(h, w, lab)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce)
    s = h.double() @ w[-500:].double().T
    full = torch.cat([torch.zeros(n, 1, dtype=torch.float64, device="cuda"), s], 1)
    full[:, 0] = torch.log(torch.tensor(v - 500.0, dtype=torch.float64))  # the zero logits, summed
    lse = torch.logsumexp(full, 1)
    label = torch.stack([s[0, 499], s[1, 100], torch.zeros((), dtype=torch.float64, device="cuda")])
    e_s = 2 * d * 2.0 ** -24 * (h.double().abs() @ w[-500:].double().abs().T).amax(1)
    close(ce.losses, lse - label, 2 * e_s + 2.0 ** -18 * (1 + lse))
    G = torch.exp(s - lse[:, None])
    G[0, 499] -= 1
    G[1, 100] -= 1
    G /= n
    e = (U[torch.bfloat16] + 2 * e_s.max().item() + 2.0 ** -18)
    close(dw[-500:], G.T @ h.double(), 1.2 * (e + U[torch.bfloat16]) * ((G.abs() + 1e-6).T @ h.double().abs()))
    close(dh, G @ w[-500:].double(), 1.2 * (e + U[torch.bfloat16] + v * 2.0 ** -23) * ((G.abs() + 1e-6) @ w[-500:].double().abs()))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("d,v", [(64, 100), (1001, 333), (4104, 5000), (12800, 301)])
def test_few_tokens(dt, n, d, v):
    """The forward that reads the weight by rows, and the products beside it."""
    h, w, lab = make(n, d, v, dt, seed=n + d)
    check(h, w, lab)
    import aethelstream_b200 as A
    from aethelstream_b200 import _lib as L
    if n > 1:
        lab[1] = IGNORE
        bad = h.clone()
        bad[1] = float("nan")
        check(bad, w, lab, ref_inputs=(h, w, lab))
    lab[0] = v
    L.device_error_bits(0)
    ce = A.cut_cross_entropy(h, w, lab)
    assert ce.losses[0].isnan() and ce.loss.isnan() and L.device_error_bits(0) == L.DEVERR_BAD_ARG
    lab[:] = IGNORE
    ce = A.cut_cross_entropy(h, w, lab)
    assert ce.loss.item() == 0 and (ce.losses == 0).all() and (ce.lse == 0).all()


@pytest.mark.parametrize("n,d,v", [(300, 2304, 5000), (2000, 2560, 3000), (1100, 8192, 1200), (600, 320, 9000)])
def test_tail_of_the_hidden_states_product(n, d, v):
    """Tile counts (of 256 x 256) that leave part of a wave, split along the vocabulary."""
    check(*make(n, d, v, torch.bfloat16, seed=d, masked=0.1))


def test_a_token_weight_that_is_not_finite():
    """It reaches its own token's gradient and d_weight, not the other tokens."""
    import aethelstream_b200 as A
    h, w, lab = make(50, 64, 300, torch.bfloat16, seed=14)
    ce = A.cut_cross_entropy(h, w, lab)
    grad = torch.rand(50, device="cuda")
    good, _ = A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=grad)
    grad[9] = 0.25 * grad.max()  # not the largest: the others' common factor stays
    good, _ = A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=grad)
    grad[9] = float("nan")
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=grad)
    others = torch.arange(50, device="cuda") != 9
    assert dh[9].isnan().all() and torch.equal(dh[others], good[others]) and dw.isnan().all()


@pytest.mark.parametrize("n", [8191, 8192, 8193, 20000])
def test_many_tokens(n):
    """Around the number of labels that one scan takes."""
    check(*make(n, 64, 300, torch.bfloat16, seed=15, masked=0.3))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [5, 40, 256, 700])
def test_gradient_of_tokens_that_are_known(n, dt):
    """Logits of 30 made of 8192 products of one sign, labels known with p = 0.999
    (a second entry close behind) or p = 1 to ten digits: G's label entry is p - 1,
    and its row adds up to zero.  A constant feature of the weight shows that sum
    in d_hidden.

    Bounds: loss and gradient make the same sums, in fp32 pieces of 512 products,
    each within c = 4e-6 of sum |h w| = S (the tensor cores' cut, up to 2.6e-6 in
    f16, and 16 additions); p of such logits is within p (1 - p) 2 c S.  lse is rounded at four
    places, and the exponentials and the logarithm are within 2^-20: p e_x.  G and
    the output are rounded once."""
    import aethelstream_b200 as A
    d, v = 8192, 600
    gen = torch.Generator(device="cuda").manual_seed(n)
    w = torch.randn(v, d, generator=gen, device="cuda") * (2.0 / d ** 0.5)
    w[250:500] = 0.77 * w[:250]
    w[:, 0] = 1.0
    w = w.to(dt)
    lab = torch.randint(0, 350, (n,), generator=gen, device="cuda")
    lab = torch.where(lab < 250, lab, lab + 250)
    h = 7.5 * w[lab].float()
    h[:, 0] = 0.0
    h = h.to(dt)
    ce = A.cut_cross_entropy(h, w, lab)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce, scale=float(n))  # every token's weight is 1
    hd, wd = h.double(), w.double()
    s = hd @ wd.T
    lse = torch.logsumexp(s, 1)
    p = torch.softmax(s, 1)
    at = lab[:, None]
    G = p.scatter_add(1, at, torch.full_like(at, -1.0, dtype=torch.float64))
    G[torch.arange(n), lab] = -(p.scatter(1, at, 0.0)).sum(1)  # p - 1 without its cancellation
    S = (hd.abs() @ wd.abs().T).amax(1, keepdim=True)
    e_x = 4 * 2.0 ** -24 * (1 + lse.abs()[:, None]) + 2.0 ** -20
    e_g = p * (1 - p) * 8e-6 * S + p * e_x + 1.1 * U[dt] * G.abs() + (2.0 ** -40 if dt is torch.float16 else 0.0)
    tiny = 2.0 ** -24 if dt is torch.float16 else 1e-38
    acc = 2 * 2.0 ** -24
    want = G @ wd
    close(dh, want, 1.1 * (e_g @ wd.abs()) + acc * v * (G.abs() @ wd.abs()) + 1.1 * U[dt] * want.abs() + tiny)
    want = G.T @ hd
    close(dw, want, 1.1 * (e_g.T @ hd.abs()) + acc * n * (G.abs().T @ hd.abs()) + 1.1 * U[dt] * want.abs() + tiny)


def hidden_bound(h, w, lab, grad, scale):
    """d_hidden in 64 bits and its bound, every token judged by its own weight (see reference())."""
    dt = h.dtype
    hd, wd = h.double(), w.double()
    s = hd @ wd.T
    g = scale * grad.double()[:, None]
    p = torch.softmax(s, 1)
    lse = torch.logsumexp(s, 1)
    e_s = (hd.abs() @ wd.abs().T).amax(1) * (2 * h.shape[1] * 2.0 ** -24)
    G = p.scatter_add(1, lab[:, None], torch.full_like(lab[:, None], -1.0, dtype=torch.float64)) * g
    e_g = G.abs() * (U[dt] + 2.0 ** -20) + (p * g.abs()) * (2 * e_s + 2.0 ** -18 * (1 + lse.abs() / 16))[:, None] + 2.0 ** -40 * g.abs()
    want = G @ wd
    return want, 1.1 * (e_g @ wd.abs()) + 2 * 2.0 ** -24 * w.shape[0] * (G.abs() @ wd.abs()) + 1.1 * U[dt] * want.abs() + 2.0 ** -24


@pytest.mark.parametrize("n,d,v", [(3, 64, 131071), (40, 64, 131071), (256, 64, 60001), (4200, 64, 40001)])
def test_token_weights_over_six_decades(n, d, v):
    """f16: a token's d_hidden has its bits whatever the other tokens weigh.  Most
    vocabulary entries are alike and their probabilities small, so that cutting
    them off would show; a constant feature shows the sum of G's row."""
    import aethelstream_b200 as A
    gen = torch.Generator(device="cuda").manual_seed(n)
    w = torch.zeros(v, d, device="cuda")
    w[:300] = torch.randn(300, d, generator=gen, device="cuda") * 0.25
    w[:, 0] = 1.0
    w = w.half()
    lab = torch.randint(0, 300, (n,), generator=gen, device="cuda")
    h = torch.randn(n, d, generator=gen, device="cuda").half()
    h[:, 0] = 0.0
    grad = torch.logspace(-6, 0, n, device="cuda")
    grad[1::2] *= -1
    scale = 2.0 ** 13
    ce = A.cut_cross_entropy(h, w, lab)
    dh, dw = A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=grad, scale=scale)
    for at in torch.arange(n, device="cuda").split(64):
        close(dh[at], *hidden_bound(h[at], w, lab[at], grad[at], scale))
    assert torch.equal(A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=grad, scale=scale, need_weight=False)[0], dh)
    assert torch.equal(A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=grad, scale=scale, need_hidden=False)[1], dw)
    if n <= 256:
        r = reference(h, w, lab, grad=grad, scale=scale)
        close(dw, r["dw"], r["b_w"])
