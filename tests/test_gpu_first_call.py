"""The first call of a process may come inside a graph's capture: nothing that
the library sets up on its first use of a device may end the capture."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SETUP = """
import sys
sys.path.insert(0, {root!r})
import torch
import aethelstream_b200 as A
gen = torch.Generator(device="cuda").manual_seed(0)
h = torch.randn(64, 256, generator=gen, device="cuda").bfloat16()
w = (0.1 * torch.randn(1000, 256, generator=gen, device="cuda")).bfloat16()
lab = torch.randint(0, 1000, (64,), generator=gen, device="cuda")
lse = torch.logsumexp(h.float() @ w.float().T, 1)
ce = A.CutCrossEntropy(lse.mean(), lse, lse)
gain = torch.ones(256, device="cuda")
ck = A.ActivationCheckpoint(torch.randint(-127, 128, (64, 256), generator=gen, device="cuda").to(torch.int8),
                            torch.full((64, 2), 0.01, device="cuda"), torch.bfloat16)

def call():
    {call}

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
for t in got:
    t.zero_()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(got, call()):
    assert torch.equal(a, b) and (a != 0).any()
print("same")
"""

CALLS = {
    "one token's loss": "c = A.cut_cross_entropy(h[:1], w, lab[:1]); return c.loss, c.losses, c.lse",
    "loss": "c = A.cut_cross_entropy(h, w, lab); return c.loss, c.losses, c.lse",
    "loss's gradient": "return A.cut_cross_entropy_backward(h, w, lab, ce)",
    "norm's gradient": "return A.rms_norm_checkpoint_backward(h, ck, gain)",
    "weight gradient": "return (A.checkpoint_weight_grad(h, ck, norm_weight=gain),)",
}


@pytest.mark.parametrize("name", CALLS)
def test_first_call_inside_a_capture(name):
    r = subprocess.run([sys.executable, "-c", SETUP.format(root=ROOT, call=CALLS[name])], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]
