"""Log probabilities at the head, entropies, alternatives and the gradient, against
their definitions in 64 bits.

Tolerances (u = 2^-8 for bf16, 2^-11 for f16, half a step relative):
  logits: fp32 sums of exact products, within 2 d 2^-24 * sum_i |h_i w_i| of the
    exact one, e_s (as the loss's test has it);
  lse and log probability: e_s twice, and 2^-18 (1 + |lse|) for the exponentials
    and the logarithm;
  entropy: d entropy / d s_v = -p_v (q_v + entropy), whose sizes add up to 2 entropy
    at most: e_s twice of that, and the same 2^-18 (1 + |lse| + entropy);
  G = a 1[y] - p (a + b (q + entropy)): relative u (rounded once; up to 128 tokens
    u^2: kept as its rounding and the rounding of what that left), the error of its
    exponent, those of q and of the entropy times p |b|, and f16's spacing beside
    the largest weight; times |W| or |H| and summed;
  outputs: rounded once more.
Which alternatives come first is compared on inputs whose products and sums are
whole numbers of one step, exact in fp32 in any order, so that equal logits are equal.
"""
import math

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


def reference(h, w, lab, a, b):
    dt = h.dtype
    n, d = h.shape
    v = w.shape[0]
    keep = lab != IGNORE
    hd = torch.where(keep[:, None], h, torch.zeros_like(h)).double()
    wd = w.double()
    s = hd @ wd.T
    lse = torch.logsumexp(s, 1)
    q = s - lse[:, None]
    p = q.exp()
    ent = -torch.where(p > 0, p * q, 0.0).sum(1)
    at = torch.where(keep, lab, 0)[:, None]
    a, b = (torch.zeros(n, dtype=torch.float64, device="cuda") if x is None else torch.where(keep, x.double(), 0.0) for x in (a, b))
    slope = a[:, None] + b[:, None] * torch.where(p > 0, q + ent[:, None], 0.0)
    G = -p * slope
    G.scatter_add_(1, at, a[:, None])
    e_s = (hd.abs() @ wd.abs().T).amax(1) * (2 * d * 2.0 ** -24)
    e_lp = 2 * e_s + 2.0 ** -18 * (1 + lse.abs())
    e_ent = 4 * e_s * ent + 2.0 ** -18 * (1 + lse.abs() + ent)
    e_g = G.abs() * ((U[dt] if n > 128 else U[dt] ** 2) + 2.0 ** -20) + p * slope.abs() * e_lp[:, None] + p * (b.abs() * (e_lp + e_ent))[:, None]
    if dt is torch.float16:
        e_g += 2.0 ** -40 * (a.abs() + (math.log(v) / 4 + 0.5) * b.abs()).max()
    dh, dw = G @ wd, G.T @ hd
    tiny = 2.0 ** -24 if dt is torch.float16 else 1e-38
    acc = 2 * 2.0 ** -24
    b_h = 1.1 * (e_g @ wd.abs()) + acc * v * (G.abs() @ wd.abs()) + 1.1 * U[dt] * dh.abs() + tiny
    b_w = 1.1 * (e_g.T @ hd.abs()) + acc * n * (G.abs().T @ hd.abs()) + 1.1 * U[dt] * dw.abs() + tiny
    zero = torch.zeros_like(lse)
    return dict(lp=torch.where(keep, q.gather(1, at)[:, 0], zero), ent=torch.where(keep, ent, zero), lse=torch.where(keep, lse, zero),
                q=q, dh=dh, dw=dw, e_lp=e_lp, e_ent=e_ent, b_h=b_h, b_w=b_w, keep=keep)


def close(got, want, bound):
    off = (got.double() - want).abs()
    assert got.isfinite().all()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def grads(n, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, generator=gen, device="cuda"), 0.3 * torch.randn(n, generator=gen, device="cuda"))


def check(h, w, lab, top=0, a=None, b=None, ref_inputs=None):
    import aethelstream_b200 as A
    if a is None and b is None:
        a, b = grads(h.shape[0], 11)
    r = A.token_log_probs(h, w, lab, top_k=top, ignore_index=IGNORE)
    dh, dw = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b, ignore_index=IGNORE)
    e = reference(*(ref_inputs or (h, w, lab)), a, b)
    close(r.log_probs, e["lp"], e["e_lp"])
    close(r.entropy, e["ent"], e["e_ent"])
    close(r.lse, e["lse"], e["e_lp"])
    close(dh, e["dh"], e["b_h"])
    close(dw, e["dw"], e["b_w"])
    if top:
        assert r.top_log_probs.shape == r.top_ids.shape == (*lab.shape, top)
        keep = e["keep"]
        assert (r.top_ids[~keep] == -1).all() and (r.top_log_probs[~keep] == 0).all()
        ids, lps = r.top_ids[keep], r.top_log_probs[keep]
        assert ((ids >= 0) & (ids < w.shape[0])).all() and (lps[:, :-1] >= lps[:, 1:]).all()
        assert (ids.sort(1).values.diff(dim=1) > 0).all()  # no entry twice
        # what they are worth, and that no other is worth more
        bound = e["e_lp"][keep][:, None]
        close(lps, e["q"][keep].gather(1, ids), bound.expand_as(lps))
        close(lps, e["q"][keep].topk(top).values, 2 * bound.expand_as(lps))
    else:
        assert r.top_log_probs is None and r.top_ids is None
    return r, dh, dw


SIZES = [(1, 64, 1000), (1, 8, 7), (2, 40, 255), (3, 136, 257), (4, 72, 5000), (5, 64, 129), (63, 512, 4099), (64, 64, 256),
         (65, 200, 513), (130, 96, 1), (255, 64, 300), (257, 1032, 700), (520, 72, 2049), (1000, 256, 77)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d,v", SIZES)
def test_sizes(dt, n, d, v):
    for top in (0, min(5, v)):
        check(*make(n, d, v, dt, seed=n + d + v), top=top)


def grid(n, d, v, dt, seed, steps):
    """Hidden states and weights of whole steps, few enough for exact sums."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randint(-steps, steps + 1, (n, d), generator=gen, device="cuda") / 8
    w = torch.randint(-steps, steps + 1, (v, d), generator=gen, device="cuda") / 16
    return h.to(dt), w.to(dt), torch.randint(0, v, (n,), generator=gen, device="cuda")


@pytest.mark.parametrize("top", [1, 2, 8, 20, 31, 32])
@pytest.mark.parametrize("n,d,v", [(1, 64, 40), (1, 256, 32000), (2, 64, 4737), (4, 512, 20000), (7, 64, 3000), (100, 64, 33),
                                   (300, 128, 4096), (700, 64, 10007), (1100, 64, 2500)])
def test_which_alternatives(n, d, v, top):
    """Indices and order, ties included: many equal logits, and few."""
    import aethelstream_b200 as A
    for steps, dt in ((1, torch.bfloat16), (16, torch.float16)):
        h, w, lab = grid(n, d, v, dt, n + v, steps)
        if steps == 1:
            w[v // 3:2 * v // 3] = w[0]  # a third of the vocabulary alike
        r = A.token_log_probs(h, w, lab, top_k=top)
        s = h.double() @ w.double().T
        want = torch.argsort(s, dim=1, descending=True, stable=True)[:, :top]
        assert torch.equal(r.top_ids, want)
        lse = torch.logsumexp(s, 1, keepdim=True)
        close(r.top_log_probs, s.gather(1, want) - lse, 2.0 ** -18 * (1 + lse.abs()).expand(n, top))


@pytest.mark.parametrize("n", [1, 3, 40, 600])
def test_all_logits_equal(n):
    import aethelstream_b200 as A
    w = torch.ones(5000, 64, device="cuda").bfloat16()
    h = torch.ones(n, 64, device="cuda").bfloat16()
    r = A.token_log_probs(h, w, torch.full((n,), 4999, device="cuda"), top_k=32)
    assert torch.equal(r.top_ids, torch.arange(32, device="cuda").expand(n, 32))
    even = math.log(5000)
    assert (r.log_probs + even).abs().max() < 2.0 ** -18 * (1 + 64 + even) and (r.entropy - even).abs().max() < 2.0 ** -18 * (1 + 64 + even)


@pytest.mark.parametrize("order", ["up", "down"])
@pytest.mark.parametrize("n", [2, 40, 500])
def test_sorted_vocabularies(n, order):
    """Logits that rise (or fall) along the whole vocabulary."""
    import aethelstream_b200 as A
    v = 20000
    w = torch.zeros(v, 64, device="cuda")
    i = torch.arange(v, device="cuda")
    w[:, 0], w[:, 1] = i // 128, i % 128  # exact in both types
    h = torch.zeros(n, 64, device="cuda")
    h[:, 0], h[:, 1] = 128 / 64, 1 / 64
    if order == "down":
        h = -h
    r = A.token_log_probs(h.bfloat16(), w.bfloat16(), i[:n], top_k=20)
    want = torch.arange(20, device="cuda")
    assert torch.equal(r.top_ids, (v - 1 - want if order == "up" else want).expand(n, 20))


def test_pieces_of_the_vocabulary():
    """More logits than a piece holds, as rows and with few live ones."""
    n, v = 4200, 40001
    h, w, lab = grid(n, 64, v, torch.bfloat16, 5, 16)
    lab[::50] = IGNORE
    r, _, _ = check(h, w, lab, top=9)
    keep = lab != IGNORE
    s = h.double() @ w.double().T
    assert torch.equal(r.top_ids[keep], torch.argsort(s, dim=1, descending=True, stable=True)[:, :9][keep])
    assert torch.equal(check(h, w, lab)[0].entropy.isfinite(), torch.ones(n, dtype=torch.bool, device="cuda"))


def test_a_large_vocabulary_of_few_tokens():
    """Pieces with tokens as the products' columns, and past what one to four keep."""
    import aethelstream_b200 as A
    v = 1000003
    for n in (1, 4, 60, 300):
        h, w, lab = grid(n, 16, v, torch.bfloat16, n, 16)
        r = A.token_log_probs(h, w, lab, top_k=8)
        s = h.double() @ w.double().T
        assert torch.equal(r.top_ids, torch.argsort(s, dim=1, descending=True, stable=True)[:, :8])
        lse = torch.logsumexp(s, 1)
        close(r.log_probs, s.gather(1, lab[:, None])[:, 0] - lse, 2.0 ** -18 * (1 + lse.abs()))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_more_tokens_than_a_scan(dt):
    """The live tokens are numbered 8192 at a time."""
    check(*make(9001, 64, 300, dt, seed=16, masked=0.3), top=4)
    check(*make(16385, 40, 70, dt, seed=17), top=2)


@pytest.mark.parametrize("top", [0, 1, 20, 32])
@pytest.mark.parametrize("n", [5, 40, 296, 297])
def test_few_tokens_of_many_ranges(n, top):
    """Eight warps a token, or one: masks, a NaN, a label outside, equal logits."""
    import aethelstream_b200 as A
    v = 66001
    h, w, lab = grid(n, 64, v, torch.bfloat16, n, 2)
    w[20000:60000] = w[7]
    h[1, 3], lab[2], lab[3] = float("nan"), IGNORE, v
    r = A.token_log_probs(h, w, lab, top_k=top)
    A._lib.device_error_bits(0)
    s = h.double() @ w.double().T
    logs = torch.log_softmax(s, 1)
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[1:4] = False
    bound = 2.0 ** -18 * (1 + torch.logsumexp(s, 1).abs())
    close(r.log_probs[good], logs.gather(1, lab.clamp(0, v - 1)[:, None])[:, 0][good], bound[good])
    close(r.entropy[good], -(logs.exp() * logs).sum(1)[good], bound[good] * 12)
    assert r.log_probs[1].isnan() and r.log_probs[2] == 0 and r.log_probs[3].isnan()
    if top:
        want = torch.argsort(s, dim=1, descending=True, stable=True)[:, :top]
        assert torch.equal(r.top_ids[good], want[good]) and (r.top_ids[1:4] == -1).all()
        close(r.top_log_probs[good], logs.gather(1, want)[good], bound[good, None].expand(-1, top))


@pytest.mark.parametrize("masked", [0.3, 0.9, 1.0])
@pytest.mark.parametrize("n", [1, 3, 40, 300, 700])
def test_masked_tokens_take_no_part(n, masked):
    h, w, lab = make(n, 128, 600, torch.bfloat16, seed=n, masked=masked)
    bad = h.clone()
    out = lab == IGNORE
    bad[out] = float("nan")
    bad[out & (torch.arange(n, device="cuda") % 2 == 0)] = float("inf")
    r, dh, dw = check(bad, w, lab, top=4, ref_inputs=(h, w, lab))
    for x in (r.log_probs, r.entropy, r.lse, dh):
        assert (x[out] == 0).all()
    if out.all():
        assert (dw == 0).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_token_weights(dt):
    """Weights over many powers of ten, zero ones, one of the two alone, no weight."""
    import aethelstream_b200 as A
    h, w, lab = make(200, 128, 1000, dt, seed=9, masked=0.1)
    a, b = grads(200, 3)
    a, b = a * torch.logspace(-3, 0, 200, device="cuda"), b * torch.logspace(0, -3, 200, device="cuda")
    a[7] = b[7] = b[8] = a[9] = 0.0
    check(h, w, lab, a=a, b=b)
    check(h, w, lab, a=a)
    check(h, w, lab, b=b)
    r = A.token_log_probs(h, w, lab)
    for dh, dw in (A.token_log_probs_backward(h, w, lab, r),
                   A.token_log_probs_backward(h, w, lab, r, grad_log_probs=torch.zeros(200, device="cuda"))):
        assert (dh == 0).all() and (dw == 0).all()
    dh, dw = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, need_weight=False)
    assert dw is None and torch.equal(dh, A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a)[0])
    dh, dw = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, need_hidden=False)
    assert dh is None and dw.isfinite().all()
    assert A.token_log_probs_backward(h, w, lab, r, need_hidden=False, need_weight=False) == (None, None)


def test_light_tokens_keep_their_gradient_in_f16():
    """A token of 1e-6 of the largest weight: its row has the bits it has alone."""
    import aethelstream_b200 as A
    h, w, lab = make(64, 128, 3000, torch.float16, seed=10)
    r = A.token_log_probs(h, w, lab)
    a, b = grads(64, 4)
    a[1:], b[1:] = 1e-6 * a[1:], 1e-6 * b[1:]
    heavy, _ = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b)
    a[0] = b[0] = 0.0
    light, _ = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b)
    assert torch.equal(heavy[1:], light[1:])


def test_gradient_against_the_losss():
    """a = -1 / n and no entropy: the cross entropy's gradient, but for the scale
    that G is held with."""
    import aethelstream_b200 as A
    h, w, lab = make(300, 128, 2000, torch.bfloat16, seed=12, masked=0.2)
    ce = A.cut_cross_entropy(h, w, lab)
    r = A.token_log_probs(h, w, lab)
    assert torch.equal(r.log_probs, -ce.losses) or (r.log_probs + ce.losses).abs().max() < 2.0 ** -18 * 20
    one = A.cut_cross_entropy_backward(h, w, lab, ce, grad_losses=torch.ones(300, device="cuda"))
    two = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=-torch.ones(300, device="cuda"))
    e = reference(h, w, lab, -torch.ones(300, device="cuda"), None)
    for x, y, bound in zip(one, two, (e["b_h"], e["b_w"])):
        assert ((x.double() - y.double()).abs() <= 2 * bound).all()


def test_gradient_against_differences():
    """d of sum(a logp + b entropy) along a direction of the hidden states."""
    import aethelstream_b200 as A
    h, w, lab = make(20, 64, 300, torch.bfloat16, seed=13)
    a, b = grads(20, 5)
    r = A.token_log_probs(h, w, lab)
    dh, _ = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b)
    z = torch.randn(20, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))

    def value(x):
        s = A.token_log_probs(x, w, lab)
        return (s.log_probs.double() * a.double() + s.entropy.double() * b.double()).sum().item()

    up, down = (h.float() + 0.05 * z).bfloat16(), (h.float() - 0.05 * z).bfloat16()
    step = (up.double() - down.double())
    # bf16 of dh: 2^-8 of each of 1280 products; third derivatives: |step / 2|^3 of logits of a size of 1 a token
    slack = (dh.double() * step).abs().sum().item() * 2.0 ** -8 + 20 * (step.abs().max().item() * 64 ** 0.5) ** 3
    assert abs(value(up) - value(down) - (dh.double() * step).sum().item()) < slack


def test_large_logits_and_lowest_entries():
    """Logits of hundreds; entries at the type's lowest value; entries at -infinity,
    which have probability 0 and come last."""
    import aethelstream_b200 as A
    check(*make(90, 64, 1500, torch.bfloat16, seed=4, scale=60.0), top=3)
    h, w, lab = make(90, 64, 1500, torch.bfloat16, seed=5)
    h[:, 0] = 1.0
    w[:, 0] = 0.0
    lab = lab % 700
    for low in (torch.finfo(torch.bfloat16).min, -float("inf")):
        w[700:, 0] = low
        for n in (1, 3, 90):
            r = A.token_log_probs(h[:n], w, lab[:n], top_k=7)
            e = reference(h[:n], w[:700], lab[:n], None, None)
            close(r.log_probs, e["lp"], e["e_lp"])
            close(r.entropy, e["ent"], e["e_ent"])
            assert (r.top_ids < 700).all()
    few = torch.full((40, 64), 0.0, device="cuda").bfloat16()
    few[5:, 0] = -float("inf")
    for n in (2, 30):
        r = A.token_log_probs(h[:n], few, lab[:n] % 5, top_k=8)
        assert torch.equal(r.top_ids, torch.arange(8, device="cuda").expand(n, 8))
        assert (r.top_log_probs[:, 5:] == -float("inf")).all() and r.entropy.isfinite().all()


@pytest.mark.parametrize("n", [3, 70, 600])
def test_a_live_token_that_is_not_finite(n):
    import aethelstream_b200 as A
    h, w, lab = make(n, 64, 500, torch.bfloat16, seed=6)
    good = A.token_log_probs(h, w, lab, top_k=6)
    h2 = h.clone()
    h2[1, 5] = float("nan")
    r = A.token_log_probs(h2, w, lab, top_k=6)
    others = torch.arange(n, device="cuda") != 1
    for x, y in ((r.log_probs, good.log_probs), (r.entropy, good.entropy), (r.lse, good.lse), (r.top_log_probs, good.top_log_probs)):
        assert x[1].isnan().all() and torch.equal(x[others], y[others])
    assert (r.top_ids[1] == -1).all() and torch.equal(r.top_ids[others], good.top_ids[others])
    a, b = grads(n, 7)
    dh, _ = A.token_log_probs_backward(h2, w, lab, r, grad_log_probs=a, grad_entropy=b)
    assert dh[1].isnan().all() and dh[others].isfinite().all()


@pytest.mark.parametrize("n", [4, 30, 600])
def test_label_outside_the_vocabulary(n):
    import aethelstream_b200 as A
    from aethelstream_b200 import _lib as L
    L.device_error_bits(0)
    h, w, lab = make(n, 64, 100, torch.bfloat16, seed=7)
    good = A.token_log_probs(h, w, lab, top_k=3)
    lab2 = lab.clone()
    lab2[1], lab2[2] = 100, -7
    r = A.token_log_probs(h, w, lab2, top_k=3)
    out = torch.zeros(n, dtype=torch.bool, device="cuda")
    out[1:3] = True
    for x, y in ((r.log_probs, good.log_probs), (r.entropy, good.entropy), (r.top_log_probs, good.top_log_probs)):
        assert x[out].isnan().all() and torch.equal(x[~out], y[~out])
    assert (r.top_ids[out] == -1).all()
    a, b = grads(n, 8)
    dh, dw = A.token_log_probs_backward(h, w, lab2, r, grad_log_probs=a, grad_entropy=b)
    assert (dh[out] == 0).all() and dh.isfinite().all() and dw.isfinite().all()
    assert L.device_error_bits(0) == L.DEVERR_BAD_ARG and L.device_error_bits(0) == 0


def test_strides_shapes_and_label_types():
    import aethelstream_b200 as A
    h, w, lab = make(24, 64, 300, torch.bfloat16, seed=8, masked=0.2)
    a, b = grads(24, 9)
    r = A.token_log_probs(h, w, lab, top_k=3)
    dh, dw = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b)
    wide = torch.randn(48, 131, device="cuda").bfloat16()
    wide[::2, 67:] = h
    ww = torch.randn(300, 70, device="cuda").bfloat16()
    ww[:, 3:67] = w
    hs, ws, ls = wide[::2, 67:].unflatten(0, (4, 6)), ww[:, 3:67], lab.int().view(4, 6)
    r2 = A.token_log_probs(hs, ws, ls, top_k=3)
    dh2, dw2 = A.token_log_probs_backward(hs, ws, ls, r2, grad_log_probs=a.view(4, 6), grad_entropy=b.view(4, 6))
    assert r2.log_probs.shape == r2.entropy.shape == (4, 6) and r2.top_ids.shape == (4, 6, 3)
    for x, y in ((r2.log_probs, r.log_probs), (r2.entropy, r.entropy), (r2.top_log_probs, r.top_log_probs), (r2.top_ids, r.top_ids)):
        assert torch.equal(x.flatten(0, 1), y)
    assert torch.equal(dh2.view(24, 64), dh) and torch.equal(dw2, dw)


@pytest.mark.parametrize("n", [1, 2, 5, 33, 127, 128, 129])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gradients_of_few_tokens(dt, n):
    """Weights just above powers of two, which 16 bits round the most: nothing evens
    that out where a token or two make up a row."""
    h, w, lab = make(n, 264, 1200, dt, seed=18, masked=0.3 if n > 5 else 0.0)
    a, b = grads(n, 19)
    a = a.sign() * (1.0 + 0.9 * U[dt])
    check(h, w, lab, a=a, b=1e-3 * b)


@pytest.mark.parametrize("n", [3, 40, 600])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_without_gradients_and_an_entry_as_the_ignored(dt, n):
    import aethelstream_b200 as A
    h, w, lab = make(n, 72, 900, dt, seed=16, masked=0.4)
    r = A.token_log_probs(h, w, lab, top_k=2)
    dh, dw = A.token_log_probs_backward(h, w, lab, r)
    assert (dh == 0).all() and (dw == 0).all()
    a, b = grads(n, 17)
    lab = torch.where(lab == 5, 6, lab)
    r = A.token_log_probs(h, w, lab, top_k=2)
    want = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b)
    other = torch.where(lab == IGNORE, 5, lab)
    s = A.token_log_probs(h, w, other, top_k=2, ignore_index=5)
    got = A.token_log_probs_backward(h, w, other, s, grad_log_probs=a, grad_entropy=b, ignore_index=5)
    for x, y in ((r.log_probs, s.log_probs), (r.entropy, s.entropy), (r.lse, s.lse), (r.top_ids, s.top_ids), *zip(want, got)):
        assert torch.equal(x, y)


def test_nothing_to_do():
    import aethelstream_b200 as A
    h, w, lab = torch.empty(0, 64, device="cuda").half(), torch.ones(10, 64, device="cuda").half(), torch.empty(0, dtype=torch.int64, device="cuda")
    r = A.token_log_probs(h, w, lab, top_k=2)
    assert r.log_probs.shape == (0,) and r.top_ids.shape == (0, 2)
    dh, dw = A.token_log_probs_backward(h, w, lab, r)
    assert dh.shape == (0, 64) and (dw == 0).all()


@pytest.mark.parametrize("n", [2, 50, 700])
def test_captured_and_repeated(n):
    """A replay follows its inputs; equal calls give equal bits, another stream too."""
    import aethelstream_b200 as A
    h, w, lab = make(n, 128, 3000, torch.bfloat16, seed=14)
    a, b = grads(n, 10)

    def call():
        r = A.token_log_probs(h, w, lab, top_k=5)
        return (r.log_probs, r.entropy, r.top_log_probs, r.top_ids,
                *A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b))

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    h.mul_(0.5)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    for x, y, z in zip(got, call(), other):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_refusals():
    import aethelstream_b200 as A
    h, w, lab = make(8, 64, 20, torch.bfloat16, seed=15)
    for bad in (dict(top_k=-1), dict(top_k=21), dict(top_k=33)):
        with pytest.raises(ValueError):
            A.token_log_probs(h, w, lab, **bad)
    for bad in ((h.float(), w.float(), lab), (h, w.half(), lab), (h, w, lab[:3]), (h, w, lab.float()), (h, w.cpu(), lab)):
        with pytest.raises(ValueError):
            A.token_log_probs(*bad)
    r = A.token_log_probs(h, w, lab)
    g = torch.ones(8, device="cuda")
    for kw in (dict(grad_log_probs=g[:3]), dict(grad_entropy=g.double()), dict(grad_log_probs=g.cpu())):
        with pytest.raises(ValueError):
            A.token_log_probs_backward(h, w, lab, r, **kw)
    r.lse = r.lse[:3]
    with pytest.raises(ValueError):
        A.token_log_probs_backward(h, w, lab, r, grad_log_probs=g)
