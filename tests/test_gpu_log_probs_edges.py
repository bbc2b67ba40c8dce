"""Log probabilities at the head where their arithmetic has an edge."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("n", [2, 40, 256, 1100])
@pytest.mark.parametrize("power,sign", [(16, 1), (20, 1), (25, -1), (25, 1), (27, 1), (31, 1), (60, -1), (100, 1)])
def test_logits_of_any_finite_size(power, sign, n, top):
    """Half of the vocabulary has the largest logit, the other half less by
    2^(power - 20), all around +-2^power.  The logits are exact in fp32, and so is
    their distance from the maximum; what is left is the error of 1500 exponentials
    of 2^-21 each, their sum and its logarithm: 2^-18 of 1 + the result covers these."""
    import aethelstream_b200 as A
    v = 1500
    h, w = torch.zeros(n, 64, device="cuda"), torch.zeros(v, 64, device="cuda")
    h[:, 0], w[:, 0] = 2.0 ** (power - power // 2), sign * 2.0 ** (power // 2)
    h[:, 1], w[1::2, 1] = 2.0 ** (power - 20), 1.0
    lab = torch.arange(n, device="cuda") % v
    r = A.token_log_probs(h.bfloat16(), w.bfloat16(), lab, top_k=top)
    s = h[:1].double() @ w.double().T
    q = torch.log_softmax(s, 1)[0]
    entropy = -(q.exp() * torch.where(q > -700, q, 0.0)).sum()
    assert ((r.entropy.double() - entropy).abs() <= 2.0 ** -18 * (1 + entropy)).all()
    assert ((r.log_probs.double() - q[lab]).abs() <= 2.0 ** -18 * (1 + q[lab].abs())).all()
    assert ((r.lse.double() - torch.logsumexp(s, 1)).abs() <= 2.0 ** -18 + 2.0 ** -23 * 2.0 ** power).all()
    if top:
        assert torch.equal(r.top_ids, torch.tensor([1, 3, 5], device="cuda").expand(n, 3))
        assert ((r.top_log_probs.double() - q[1]).abs() <= 2.0 ** -18 * (1 + q[1].abs())).all()


def test_results_are_tensors_of_their_own():
    """Log probabilities changed in place (for a ratio to older ones, say) leave what the
    backward pass saved as it is, and torch agrees."""
    import aethelstream_b200 as A

    class LogProbs(torch.autograd.Function):
        @staticmethod
        def forward(ctx, h, w, lab):
            r = A.token_log_probs(h, w, lab)
            ctx.save_for_backward(h, w, lab, r.lse, r.entropy)
            ctx.result = r
            return r.log_probs

        @staticmethod
        def backward(ctx, g):
            h, w, lab, lse, entropy = ctx.saved_tensors
            r = A.TokenLogProbs(None, entropy, lse, None, None)
            return *A.token_log_probs_backward(h, w, lab, r, grad_log_probs=g.contiguous()), None

    gen = torch.Generator(device="cuda").manual_seed(1)
    h, w = (torch.randn(n, 64, generator=gen, device="cuda").bfloat16().requires_grad_() for n in (20, 300))
    lab = torch.arange(20, device="cuda")
    old = torch.randn(20, generator=gen, device="cuda")
    LogProbs.apply(h, w, lab).sub_(old).sum().backward()
    r = A.token_log_probs(h.detach(), w.detach(), lab)
    dh, dw = A.token_log_probs_backward(h.detach(), w.detach(), lab, r, grad_log_probs=torch.ones(20, device="cuda"))
    assert torch.equal(h.grad, dh) and torch.equal(w.grad, dw)


@pytest.mark.parametrize("live", [1, 2, 40, 128, 129])
@pytest.mark.parametrize("n", [129, 200, 256, 300, 700, 1100, 8192, 9001])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_a_padded_batch_has_the_gradient_of_its_tokens(dt, n, live):
    """As test_gradients_of_few_tokens, within its bounds (u^2 for G up to 128 tokens),
    with the tokens anywhere among others that take no part."""
    import aethelstream_b200 as A
    from test_gpu_log_probs import IGNORE, U, close, grads, make, reference
    h, w, lab = make(n, 264, 1200, dt, seed=n + live)
    a, b = grads(n, 19)
    a, b = a.sign() * (1.0 + 0.9 * U[dt]), 1e-3 * b
    gen = torch.Generator(device="cuda").manual_seed(n)
    keep = torch.zeros(n, dtype=torch.bool, device="cuda")
    keep[torch.randperm(n, generator=gen, device="cuda")[:live]] = True
    e = reference(h[keep], w, lab[keep], a[keep], b[keep])
    lab[~keep], h[~keep], a[~keep] = IGNORE, float("nan"), float("inf")
    r = A.token_log_probs(h, w, lab)
    close(r.entropy[keep], e["ent"], e["e_ent"])
    dh, dw = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b)
    close(dh[keep], e["dh"], e["b_h"])
    close(dw, e["dw"], e["b_w"])
    assert (dh[~keep] == 0).all()
    # the same where only one of the two is wanted
    one = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b, need_weight=False)[0]
    two = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=a, grad_entropy=b, need_hidden=False)[1]
    assert torch.equal(one, dh)
    close(two, e["dw"], e["b_w"])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,live", [(3, 3), (20, 15), (300, 290)])
@pytest.mark.parametrize("of", ["both", "log probabilities", "entropy"])
def test_gradients_against_differences_in_64_bits(of, dt, n, live):
    """Slopes of sum(a logp + b entropy) from values on both sides, in 64 bits: along
    random directions and along the gradients themselves, where no sum cancels.

    Half steps of 2^-12 of directions of length 1: the third derivative's part is below
    1e-6 of a slope (logits change by 2^-12 |W| = 1e-3 at most), 64 bits' own rounding
    below 1e-9.  A gradient's element is off by its rounding u and as much again where G
    is rounded once (129 tokens on), which adds up along a direction z to 2 u sum |g z|
    at most where all of G's error goes one way: along the gradient 2 u of the slope."""
    import aethelstream_b200 as A
    from test_gpu_log_probs import IGNORE, U, grads, make
    h, w, lab = make(n, 64, 300, dt, seed=13)
    lab[live:] = IGNORE
    a, b = grads(n, 5)
    r = A.token_log_probs(h, w, lab)
    got = A.token_log_probs_backward(h, w, lab, r, grad_log_probs=None if of == "entropy" else a,
                                     grad_entropy=None if of == "log probabilities" else b)
    a, b = a * (of != "entropy"), b * (of != "log probabilities")

    def value(x, y):
        q = torch.log_softmax(x[:live] @ y.T, 1)
        lp = q.gather(1, lab[:live, None])[:, 0]
        return (lp * a[:live].double() - b[:live].double() * (q.exp() * q).sum(1)).sum().item()

    gen = torch.Generator(device="cuda").manual_seed(6)
    for which, x in enumerate((h, w)):
        g = got[which].double()
        for along in (False, False, False, True):
            z = g.clone() if along else torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
            z /= z.norm()
            at = [h.double(), w.double()]
            ends = []
            for sign in (1, -1):
                at[which] = x.double() + sign * 2.0 ** -12 * z
                ends.append(value(*at))
            slope = (ends[0] - ends[1]) * 2.0 ** 11
            slack = 2.2 * U[dt] * (g * z).abs().sum().item() + 1e-5 * abs(slope) + 1e-8
            assert abs(slope - (g * z).sum().item()) <= slack, (which, along)
            assert not along or slack < abs(slope) / 50
    assert (got[0][live:] == 0).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d,v", [(1, 1, 1), (1, 3, 2), (3, 1, 2), (4, 33, 129), (5, 3, 1), (40, 7, 600), (129, 1, 3), (130, 65, 257), (257, 5, 2),
                                   (300, 129, 1001), (513, 31, 40), (1100, 13, 300)])
def test_odd_features_and_single_entries(dt, n, d, v):
    from test_gpu_log_probs import check, make
    for masked in (0.0, 0.6):
        h, w, lab = make(n, d, v, dt, seed=n + d + v, masked=masked)
        check(h, w, lab, top=min(3, v))
        check(h.view(1, n, 1, d).expand(2, n, 1, d)[1, :, 0], w.repeat(1, 2)[:, d:], lab)  # rows off 16 bytes


@pytest.mark.parametrize("top", [16, 20, 32])
@pytest.mark.parametrize("n", [5, 40, 296, 297])
def test_many_alternatives_of_many_ranges(n, top):
    """Eight warps a token with as many alternatives as there are, or one: equal logits
    by the thousand, masks, a NaN; indices and their order exact."""
    import aethelstream_b200 as A
    from test_gpu_log_probs import IGNORE, close, grid
    v = 140001
    h, w, lab = grid(n, 64, v, torch.bfloat16, n, 2)
    w[20000:60000] = w[7]
    h[1, 3], lab[2] = float("nan"), IGNORE
    r = A.token_log_probs(h, w, lab, top_k=top)
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[1:3] = False
    logs = torch.log_softmax(h.double() @ w.double().T, 1)
    want = torch.argsort(logs, dim=1, descending=True, stable=True)[:, :top]
    assert torch.equal(r.top_ids[good], want[good]) and (r.top_ids[1:3] == -1).all()
    assert r.top_log_probs[1].isnan().all() and (r.top_log_probs[2] == 0).all()
    bound = 2.0 ** -18 * (20 + logs.gather(1, want).abs())
    close(r.top_log_probs[good], logs.gather(1, want)[good], bound[good])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 4, 40, 256, 1100])
def test_no_log_probability_above_zero_and_no_entropy_below(dt, n):
    """Distributions of one entry, and nearly so, where a sum's rounding is all there is."""
    import aethelstream_b200 as A
    gen = torch.Generator(device="cuda").manual_seed(n)
    for v, scale in ((1, 1.0), (1, 100.0), (2, 8.0), (129, 8.0), (5000, 12.0)):
        h = (scale * torch.randn(n, 64, generator=gen, device="cuda")).to(dt)
        w = torch.randn(v, 64, generator=gen, device="cuda").to(dt)
        lab = (h.float() @ w.float().T).argmax(1)
        top = min(3, v)
        for r in (A.token_log_probs(h, w, lab), A.token_log_probs(h, w, lab, top_k=top)):
            assert (r.log_probs <= 0).all() and (r.entropy >= 0).all(), (v, r.log_probs.max().item(), r.entropy.min().item())
        assert (r.top_log_probs <= 0).all()
