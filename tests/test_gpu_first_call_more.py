"""The first call of a process inside a graph's capture, for the operators of queries
and keys and the log probabilities."""
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
logs = torch.log_softmax(h.float() @ w.float().T, 1)
r = A.TokenLogProbs(logs[:, 0], -(logs.exp() * logs).sum(1), torch.logsumexp(h.float() @ w.float().T, 1), None, None)
g = torch.randn(64, generator=gen, device="cuda")
q, k, gain, pos, plan = h.view(64, 4, 64), h.view(64, 4, 64)[:, :1], torch.ones(64, device="cuda"), torch.arange(64, device="cuda"), A.RotaryPlan(64, device="cuda")

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
    "one token": "c = A.token_log_probs(h[:1], w, lab[:1], top_k=4); return c.log_probs, c.entropy, c.top_log_probs, c.top_ids",
    "tokens": "c = A.token_log_probs(h, w, lab, top_k=4); return c.log_probs, c.entropy, c.top_log_probs, c.top_ids",
    "their gradient": "return A.token_log_probs_backward(h, w, lab, r, grad_log_probs=g, grad_entropy=g)",
    "rotation": "return A.rotary(q, k, pos, plan)",
    "norms": "return A.qk_norm_rotary(q, k, gain, gain, pos, plan)",
    "norms' gradient": "return A.qk_norm_rotary_backward(q, k, q, k, gain, gain, pos, plan)",
}


@pytest.mark.parametrize("name", CALLS)
def test_first_call_inside_a_capture(name):
    r = subprocess.run([sys.executable, "-c", SETUP.format(root=ROOT, call=CALLS[name])], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]
