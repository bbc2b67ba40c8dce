"""Norms of queries and keys where squares and cubes of a row's size leave fp32.

Tolerances as in test_gpu_qk.py: u = 2^-24, a turned feature 8 u of its pair's two
parts, the norm's factor (d / 2 + 8) u, the mean's d products and its factors
4 (d + 16) u of the two terms that dx is made of; half a step of the result's type.
"""
import pytest
import torch

from test_gpu_qk import U, close, norm, turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power,eps", [(30, 1e-6), (45, 1e-6), (56, 1e-6), (-30, 0.0), (-45, 0.0), (-56, 0.0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,hq,hk,d,r", [(33, 8, 2, 128, 128), (33, 3, 1, 96, 64), (21, 6, 2, 80, 40), (9, 2, 1, 200, 96), (6, 2, 1, 513, 512)])
def test_gradient_of_large_and_small_rows(n, hq, hk, d, r, dtype, power, eps):
    """Both terms of dx are of the size 1 / |x| times the gradient's."""
    import aethelstream_b200 as A
    gen = torch.Generator(device="cuda").manual_seed(d + power)
    plan = A.RotaryPlan(r, device="cuda")
    pos = torch.randint(0, 1 << 17, (n,), generator=gen, device="cuda")
    q, k = ((2.0 ** power * torch.randn(n, h, d, generator=gen, device="cuda")).to(dtype) for h in (hq, hk))
    dq, dk = (torch.randn(n, h, d, generator=gen, device="cuda").to(dtype) for h in (hq, hk))
    wq, wk = (1 + 0.1 * torch.randn(d, generator=gen, device="cuda") for _ in range(2))
    out = A.qk_norm_rotary(q, k, wq, wk, pos, plan, eps=eps)
    got = A.qk_norm_rotary_backward(dq, dk, q, k, wq, wk, pos, plan, eps=eps)
    for x, w, y, dy, dx, dw in ((q, wq, out[0], dq, got[0], got[2]), (k, wk, out[1], dk, got[1], got[3])):
        x, w = x.double(), w.double()
        want, slack = turn(plan, norm(x, w, eps)[0], pos)
        close(y, want, slack + (d / 2 + 8) * U * (want.abs() + want.abs().amax(-1, keepdim=True)), "forward")
        g, gs = turn(plan, dy.double(), pos, -1.0)
        rr = norm(x, w, eps)[1]
        z = x * rr  # of size 1
        mean = (w * g * z).mean(-1, keepdim=True)
        want = rr * (w * g - z * mean)
        slack = rr * (w.abs() * gs + z.abs() * (w.abs() * gs * z.abs()).mean(-1, keepdim=True))
        slack = slack + 4 * (d + 16) * U * rr * ((w * g).abs() + z.abs() * (w * g * z).abs().mean(-1, keepdim=True))
        close(dx, want, slack, "dx")
        terms = g * z
        ws = (gs * z.abs()).sum((0, 1)) + (n * x.shape[1] + d + 16) * U * terms.abs().sum((0, 1))
        close(dw, terms.sum((0, 1)), ws, "dw")
