"""GPU: the very first call of a kernel in a process may be the one that is captured: its workspace, its limit on LDS and its
share of the GPU are found without an eager call before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
import graphsage_amd as gs
x0 = torch.randn(8, 8, device="cuda")
torch.cuda.synchronize()
side = torch.cuda.Stream()
for M, F, dtype in ((500, 64, torch.float32), (300, 1024, torch.bfloat16), (200, 5120, torch.bfloat16), (70, 6000, torch.float32),
                    (50, 16_000, torch.float32), (20, 20_000, torch.float16)):
    x = torch.randn(M, F, device="cuda").to(dtype).requires_grad_()
    w = torch.ones(F, device="cuda").requires_grad_()
    g = torch.randn(M, F, device="cuda").to(dtype)
    seed = torch.tensor([5], device="cuda")

    def step():
        y = gs.dropout_add_layer_norm(x, None, w, p=0.3, seed=seed)
        return [y.detach(), *torch.autograd.grad(y, [x, w], g)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        seed.fill_(i + 7)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), (M, F, i)
        torch.cuda.synchronize()
    print("ok", M, F, flush=True)
"""


def test_capture_without_a_call_before():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", SCRIPT], cwd=root, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and run.stdout.count("ok") == 6, run.stdout + run.stderr
