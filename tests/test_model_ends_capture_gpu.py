"""The first call of a process may be one that is captured: nothing is set up, loaded or allocated on the side."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch
from raf_b200 import op

g = torch.Generator(device="cuda").manual_seed(0)
x, ids = torch.randn(500, 64, generator=g, device="cuda"), torch.randint(0, 500, (6000,), generator=g, device="cuda")
few = ids[:100].clone()
pred = torch.randn(40, 20000, generator=g, device="cuda")
teacher, classes = torch.randn(40, 8, generator=g, device="cuda"), torch.randint(0, 20000, (40, 8), generator=g, device="cuda")

def step():
    y, loss = op.embedding(x, ids), op.distill_loss(pred, teacher, classes)
    return [y, op.embedding_dx(y, ids, 500), op.embedding_dx(y[:100], few, 500), *loss, op.distill_loss_dpred(None, pred, teacher, classes, loss[1]),
            *op.distill_loss_with_dpred(None, pred, teacher, classes), *op.distill_loss_with_dpred(None, pred[:, :900].contiguous(), teacher, classes)]

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
for k in range(2):
    for t in (x, pred, teacher):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
print("as captured")
"""


def test_a_process_that_begins_with_a_capture():
    r = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as captured" in r.stdout, r.stdout + r.stderr
