"""A policy-gradient step of a small attention block that uses the operators
together, as a training program does: norms of queries and keys with the rotation,
log probabilities and entropy at the head, their gradients back through the block,
and one AdamW step of every parameter, against the same step in 64 bits.  Then the
generation of one token after the other with the block that was trained.

Tolerances: every activation and gradient passes through bf16 (2^-9 of itself on
average) a dozen times, which leaves some 1 % of a gradient's norm; 4 % are allowed.
AdamW's first step is a sign, so it is compared at the gradients that it was given."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

V, D, H, K, HD, T, BATCH = 1003, 256, 4, 2, 64, 48, 3
EPS = 1e-6


@pytest.fixture(scope="module")
def A():
    import aethelstream_b200
    return aethelstream_b200


def parameters():
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return {"embed": rand(V, D).bfloat16(), "qkv": (rand((H + 2 * K) * HD, D) * D ** -0.5).bfloat16(),
            "out": (rand(D, H * HD) * (H * HD) ** -0.5).bfloat16(), "head": (rand(V, D) * D ** -0.5).bfloat16(),
            "q_gain": 1 + 0.1 * rand(HD), "k_gain": 1 + 0.1 * rand(HD)}


def attention(q, k, v, mask):
    """Plain causal attention of (batch, tokens, heads, features), keys and values shared by H / K heads."""
    k, v = (x.repeat_interleave(H // K, 2) for x in (k, v))
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(HD)
    return torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(mask, -float("inf")), -1), v)


class Step:
    def __init__(self, A):
        self.A, self.p = A, parameters()
        self.plan = A.RotaryPlan(HD, layout="half", scaling="yarn", factor=4.0, original_length=32, device="cuda")
        self.names = list(self.p)
        self.state = A.AdamWState.zeros(self.p.values(), bits=8, master=True)
        self.config = A.AdamWConfig(lr=1e-3, weight_decay=0.1, beta2=0.95)

    def forward(self, ids):
        A, p = self.A, self.p
        x = p["embed"][ids]
        qkv = (x @ p["qkv"].T).view(*ids.shape, H + 2 * K, HD)
        q, k, v = qkv.split([H, K, K], 2)
        pos = torch.arange(ids.shape[1], device="cuda")
        qr, kr = A.qk_norm_rotary(q, k, p["q_gain"], p["k_gain"], pos, self.plan, eps=EPS)
        return x, q, k, v, pos, qr, kr

    def gradients(self, ids, labels, advantage, bonus):
        """Gradients of sum(advantage logp + bonus entropy), by the operators; attention's and the products' by autograd."""
        A, p = self.A, self.p
        x, q, k, v, pos, qr, kr = self.forward(ids)
        mask = torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1)
        qr, kr, v = (t.detach().requires_grad_(True) for t in (qr, kr, v))
        y = attention(qr.float(), kr.float(), v.float(), mask).flatten(2).bfloat16()
        h = x + y.detach() @ p["out"].T
        r = A.token_log_probs(h, p["head"], labels, top_k=3)
        dh, d_head = A.token_log_probs_backward(h, p["head"], labels, r, grad_log_probs=advantage, grad_entropy=bonus)
        d_out = dh.flatten(0, 1).T @ y.detach().flatten(0, 1)
        y.backward(dh @ p["out"])
        dq, dk, d_qg, d_kg = A.qk_norm_rotary_backward(qr.grad, kr.grad, q, k, p["q_gain"], p["k_gain"], pos, self.plan, eps=EPS)
        d_qkv_rows = torch.cat([dq, dk, v.grad], 2).flatten(2)
        d_qkv = d_qkv_rows.flatten(0, 1).T @ x.flatten(0, 1)
        dx = dh + d_qkv_rows @ p["qkv"]
        d_embed = torch.zeros(V, D, device="cuda").index_add_(0, ids.flatten(), dx.flatten(0, 1).float())
        return r, {"embed": d_embed, "qkv": d_qkv, "out": d_out, "head": d_head, "q_gain": d_qg, "k_gain": d_kg}

    def update(self, grads, clip):
        self.A.adamw_step([self.p[n] for n in self.names], [grads[n] for n in self.names], self.state, self.config, clip=clip,
                          decay=["gain" not in n for n in self.names])


def reference(p, ids, labels, advantage, bonus, plan):
    """The same in 64 bits: log probabilities, entropies and the parameters' gradients."""
    p = {n: t.double().requires_grad_(True) for n, t in p.items()}
    x = p["embed"][ids]
    q, k, v = (x @ p["qkv"].T).view(*ids.shape, H + 2 * K, HD).split([H, K, K], 2)
    angle = torch.arange(T, device="cuda").double()[:, None, None] * torch.tensor(plan.inv_freq, device="cuda", dtype=torch.float64)
    c, s = plan.amplitude * torch.cos(angle), plan.amplitude * torch.sin(angle)

    def through(t, gain):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * gain
        u, w = t.chunk(2, -1)
        return torch.cat([u * c - w * s, w * c + u * s], -1)

    mask = torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1)
    h = x + attention(through(q, p["q_gain"]), through(k, p["k_gain"]), v, mask).flatten(2) @ p["out"].T
    logs = torch.log_softmax(h @ p["head"].T, -1)
    keep = labels >= 0
    lp = logs.gather(2, labels.clamp(min=0)[..., None])[..., 0]
    entropy = -(logs.exp() * logs).sum(-1)
    (torch.where(keep, lp, 0) * advantage.double() + torch.where(keep, entropy, 0) * bonus.double()).sum().backward()
    return torch.where(keep, lp, 0).detach(), torch.where(keep, entropy, 0).detach(), {n: t.grad for n, t in p.items()}


def batch():
    gen = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(0, V, (BATCH, T), generator=gen, device="cuda")
    labels = torch.randint(0, V, (BATCH, T), generator=gen, device="cuda")
    labels[:, :7] = -100  # a prompt
    labels[2, 30:] = -100  # a shorter answer
    advantage = torch.randn(BATCH, T, generator=gen, device="cuda") / T
    return ids, labels, advantage, torch.full((BATCH, T), 0.01, device="cuda")


def test_a_step(A):
    step, (ids, labels, advantage, bonus) = Step(A), batch()
    clip = torch.tensor(0.5, device="cuda")
    for number in (1, 2):
        before = {n: t.clone() for n, t in step.p.items()}
        r, got = step.gradients(ids, labels, advantage, bonus)
        lp, entropy, want = reference(step.p, ids, labels, advantage, bonus, step.plan)
        assert (r.log_probs.double() - lp).abs().max() < 0.1 and (r.entropy.double() - entropy).abs().max() < 0.1
        assert (r.log_probs.double() - lp).norm() < 0.01 * lp.norm()
        for n, g in want.items():
            assert (got[n].double() - g).norm() < 0.04 * g.norm(), n
        master, m, v = step.state.master.double(), *(t.double() for t in A.adamw_moments(step.state))
        step.update(got, clip)
        at = 0
        for n in step.names:  # the formula at these gradients, from the state before
            p, size = before[n], before[n].numel()
            span = slice(at, at + size)
            g = 0.5 * got[n].double().flatten()
            m1, v1 = 0.9 * m[span] + 0.1 * g, 0.95 * v[span] + 0.05 * g * g
            u = m1 / (1 - 0.9 ** number) / ((v1 / (1 - 0.95 ** number)).sqrt() + 1e-8) + (0.1 if "gain" not in n else 0.0) * master[span]
            new = master[span] - 1e-3 * u
            assert (step.state.master[span].double() - new).abs().max() < 1e-7 + 2 ** -23 * new.abs().max(), n
            assert torch.equal(step.p[n].flatten(), step.state.master[span].to(p.dtype))
            at += -(-size // 2048) * 2048
    assert int(step.state.step) == 2


def test_a_captured_step(A):
    """The whole step's operators in a graph: replayed twice, as two steps."""
    ids, labels, advantage, bonus = batch()
    clip = torch.tensor(0.5, device="cuda")
    h = torch.randn(BATCH * T, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).bfloat16()
    results = []
    for captured in (False, True):
        step = Step(A)
        p = step.p
        qkv = (h @ p["qkv"].T).view(BATCH * T, H + 2 * K, HD)
        pos = torch.arange(BATCH * T, device="cuda")

        def once():
            q, k = A.qk_norm_rotary(qkv[:, :H], qkv[:, H:H + K], p["q_gain"], p["k_gain"], pos, step.plan)
            *_, d_qg, d_kg = A.qk_norm_rotary_backward(q, k, qkv[:, :H], qkv[:, H:H + K], p["q_gain"], p["k_gain"], pos, step.plan)
            r = A.token_log_probs(h, p["head"], labels.flatten(), top_k=2)
            _, d_head = A.token_log_probs_backward(h, p["head"], labels.flatten(), r, grad_log_probs=advantage.flatten(),
                                                   grad_entropy=bonus.flatten(), need_hidden=False)
            grads = {"embed": None, "qkv": None, "out": None, "head": d_head, "q_gain": d_qg, "k_gain": d_kg}
            step.update(grads, clip)
            return r.log_probs, r.top_ids

        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = once()
            graph.replay()
            graph.replay()
        else:
            once()
            out = once()
        results.append([*(x.clone() for x in out), *(t.clone() for t in p.values()), step.state.m.clone(), step.state.step.clone()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_one_token_after_the_other(A):
    """A generation's tokens, one call each, are those of the batch."""
    step, (ids, labels, *_) = Step(A), batch()
    x, q, k, v, pos, qr, kr = step.forward(ids[:1])
    r = A.token_log_probs(x, step.p["head"], labels[:1], top_k=5)
    for t in (0, 1, 17, T - 1):
        q1, k1 = A.qk_norm_rotary(q[:, t:t + 1], k[:, t:t + 1], step.p["q_gain"], step.p["k_gain"], pos[t:t + 1], step.plan)
        assert torch.equal(q1[0, 0], qr[0, t]) and torch.equal(k1[0, 0], kr[0, t])
        one = A.token_log_probs(x[:, t], step.p["head"], labels[:1, t], top_k=5)
        # another order of the sums: 2^-18 of logits of a size of 1
        assert (one.log_probs - r.log_probs[0, t]).abs().max() < 1e-4 and (one.entropy - r.entropy[0, t]).abs().max() < 1e-4
        if labels[0, t] >= 0:
            assert (one.top_log_probs - r.top_log_probs[0, t]).abs().max() < 1e-4


def test_two_streams_at_once(A):
    """Calls that run beside one another give what they give alone."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    plan = A.RotaryPlan(HD, device="cuda")
    w = torch.randn(HD, device="cuda", generator=gen)
    head = (0.05 * torch.randn(5000, D, device="cuda", generator=gen)).bfloat16()

    def case(n):
        q, dq = (torch.randn(n, H, HD, device="cuda", generator=gen).bfloat16() for _ in range(2))
        h = torch.randn(n, D, device="cuda", generator=gen).bfloat16()
        labels = torch.randint(0, 5000, (n,), device="cuda", generator=gen)
        params, grads = [[torch.randn(x, device="cuda", generator=gen).bfloat16() for x in (50000, 77)] for _ in range(2)]
        return q, dq, h, labels, torch.arange(n, device="cuda"), params, grads

    def run(c):
        q, dq, h, labels, pos, params, grads = c
        params = [p.clone() for p in params]
        states = [A.AdamWState.zeros(params, bits=bits) for bits in (8, 32)]
        out = []
        for _ in range(5):
            out += A.qk_norm_rotary_backward(dq, None, q, None, w, None, pos, plan)[::2]
            r = A.token_log_probs(h, head, labels, top_k=6)
            out += [r.log_probs, r.entropy, r.top_ids, *A.token_log_probs_backward(h, head, labels, r, r.entropy, r.lse)]
            for state in states:
                A.adamw_step(params, grads, state)
        return out + params + [states[0].m, states[0].v_scales, states[1].v]

    cases = [case(n) for n in (3, 300, 1111)]
    alone = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    both = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            both.append(run(c))
    torch.cuda.synchronize()
    for x, y in zip(alone, both):
        assert all(torch.equal(a, b) for a, b in zip(x, y))
