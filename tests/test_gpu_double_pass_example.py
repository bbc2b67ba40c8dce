"""The example that runs the training operators and the optimizer together: its
gradients against differentiation in 64 bits, and its loss over some steps."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("double_pass_step", os.path.join(ROOT, "examples", "double_pass_step.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_loss_falls(example):
    losses = example.train(steps=10)
    assert all(b < a for a, b in zip(losses, losses[1:])), losses
    assert losses[-1] < losses[0] - 0.5


def test_gradients_of_a_step(example, monkeypatch):
    """The weights' gradients that reach the optimizer and the gains' updates,
    against autograd of the same model in 64 bits.  Every activation and
    gradient passes through 16 bits and the norms' inputs through 8 (steps of
    1/127 of a block's maximum): a few per cent."""
    model = example.Model(256, 2, 1025, 32, 1.0)
    gen = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.randint(0, 1025, (300,), generator=gen, device="cuda")
    labels = (ids * 7 + 3) % 1025
    labels[::5] = -100
    weights = [example.A.nf4_dequantize(w, torch.float32).view(256, 256).double().requires_grad_(True) for w in model.weights]
    gains = [g.double().clone().requires_grad_(True) for g in model.gains]
    x = model.embed[ids].double()
    norm = lambda v, g: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * g  # noqa: E731
    y = norm(x, gains[0])
    for b in range(2):
        x = x + y @ weights[b].T
        y = norm(x, gains[b + 1])
    loss = torch.nn.functional.cross_entropy(y @ model.head.double().T, labels)
    loss.backward()
    seen = {}
    monkeypatch.setattr(model.opt, "project_layer", lambda keys, grads: seen.update(zip(keys, grads)))
    monkeypatch.setattr(model.opt, "finish_step", lambda *a: None)
    before = [g.clone() for g in model.gains]
    got = model.step(ids, labels, 1)
    want = float(loss.detach())
    assert abs(float(got) - want) < 0.02 * want
    for b in range(2):
        want = weights[b].grad
        assert (seen[(b, "d_wo")].double() - want).norm() < 0.05 * want.norm()
    for g, old, want in zip(model.gains, before, gains):
        assert ((old - g).double() - want.grad).norm() < 0.05 * want.grad.norm()
    model.opt.close()
