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
