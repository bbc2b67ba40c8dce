"""AdamW at the ends of its numbers' range; the formula and its bounds are those of
test_gpu_adamw.py."""
import pytest
import torch

from test_gpu_adamw import A, Check, maps, tensors  # noqa: F401 - fixtures

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [1e19, 5e19, 3e20])
def test_second_moments_next_to_the_largest_number(A, maps, kind, bits, size):  # noqa: F811
    """g^2 / 1000 still is a float, the corrected second moment no longer: the step
    is of the size of the rate all the same."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    sizes = [4096, 100]
    params = tensors(gen, sizes, [kind] * 2)
    state = A.AdamWState.zeros(params, bits=bits)
    c = Check(A, params, state, A.AdamWConfig(beta2=0.999, lr=1e-2, weight_decay=0.1), maps)
    for _ in range(2):
        c.step([(size * (0.5 + torch.rand(n, generator=gen, device="cuda"))).to(kind) for n in sizes])


@pytest.mark.parametrize("eps", [1e-10, 1e-12, 1e-15, 0.0])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind,master", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False), (torch.float16, False)])
def test_any_eps(A, maps, monkeypatch, kind, master, bits, eps):  # noqa: F811
    """Gradients from 1e-22 on, whose second moments are subnormal numbers or 0, with
    an eps beside which they count, in lists of one type.  Without eps the formula
    divides by 0 and has infinities and NaN; a NaN equals a NaN here."""
    monkeypatch.setattr(torch, "equal", lambda a, b: a.dtype == b.dtype and torch.allclose(a, b, rtol=0, atol=0, equal_nan=True))
    gen = torch.Generator(device="cuda").manual_seed(2)
    sizes = [5000, 4096, 4096, 4096, 33]
    gk = torch.float32 if kind is torch.float16 else kind
    params = tensors(gen, sizes, [kind] * 5)
    state = A.AdamWState.zeros(params, bits=bits, master=master)
    c = Check(A, params, state, A.AdamWConfig(beta1=0.9, beta2=0.999, eps=eps, lr=1e-3, weight_decay=0.1), maps)
    for _ in range(3):
        c.step([(s * torch.randn(n, generator=gen, device="cuda")).to(gk) for n, s in zip(sizes, (1e-3, 1e-19, 1e-20, 1e-22, 1e-18))])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tied_tensor_that_is_left_out(A, bits):  # noqa: F811
    """The same tensor twice, one of them without a gradient, which is not written."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    p, other, g = tensors(gen, [5000] * 3, [torch.bfloat16] * 3)
    for grads in ([g, None, None], [None, g, None]):
        both, alone = [p.clone()] * 2 + [other.clone()], p.clone()
        s, t = A.AdamWState.zeros(both, bits=bits), A.AdamWState.zeros([alone], bits=bits)
        for _ in range(2):
            A.adamw_step(both, grads, s)
            A.adamw_step([alone], [g], t)
        at = 0 if grads[0] is not None else 3
        assert torch.equal(both[0], alone) and torch.equal(both[2], other)
        assert torch.equal(s.m.view(-1, 2048)[at:at + 3], t.m.view(-1, 2048)) and int(s.step) == 2
        with pytest.raises(ValueError, match="share memory"):
            A.adamw_step(both, [g, g, None], s)
        assert int(s.step) == 2
