"""The first call of a process may be one that is captured: nothing is set up, loaded or allocated on the side.  Forward and
backward by autograd are captured together, unless an eager graph of the same leaves stands in the way."""
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


BACKWARD = """
import torch
from raf_b200 import op

g = torch.Generator(device="cuda").manual_seed(0)
table = torch.randn(500, 500, generator=g, device="cuda", requires_grad=True)
ids = torch.randint(0, 500, (60,), generator=g, device="cuda")
teacher, classes = torch.randn(60, 8, generator=g, device="cuda"), torch.randint(0, 500, (60, 8), generator=g, device="cuda")
other = torch.randn(60, 500, generator=g, device="cuda", requires_grad=True)

def step():
    table.grad = None
    loss = op.distill_loss(op.embedding(table, ids), teacher, classes)[0]
    loss.sum().backward()
    return loss.detach(), table.grad

def refused(f):
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            f()
    except RuntimeError as e:
        assert "still lives" in str(e), e
    else:
        raise SystemExit("was not refused")

logits, loss = op.embedding(table, ids), op.distill_loss(other, teacher, classes)[0]
refused(lambda: op.embedding(table, ids))
refused(lambda: op.distill_loss(logits, teacher, classes))
refused(lambda: op.distill_loss(other, teacher, classes))
with torch.cuda.graph(torch.cuda.CUDAGraph()):  # without a gradient
    op.embedding(table.detach(), ids)
    with torch.no_grad():
        op.distill_loss(other, teacher, classes)
del logits, loss

side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    step()
torch.cuda.current_stream().wait_stream(side)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
for k in range(2):
    for t in (table.data, teacher):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    ids.copy_(torch.randint(0, 500, (60,), generator=g, device="cuda"))
    graph.replay()
    got_now = [t.clone() for t in got]
    for a, b in zip(got_now, step()):
        assert torch.equal(a, b)
print("as captured")
"""


def test_a_captured_backward():
    r = subprocess.run([sys.executable, "-c", BACKWARD], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as captured" in r.stdout, r.stdout + r.stderr


WITHOUT = """
import torch
from raf_b200 import _lib, op

_lib._ops = _lib._GeneralWay()
table = torch.randn(500, 500, device="cuda", requires_grad=True)
ids = torch.randint(0, 500, (60,), device="cuda")
teacher, classes = torch.randn(60, 8, device="cuda"), torch.randint(0, 500, (60, 8), device="cuda")
logits = torch.randn(60, 500, device="cuda", requires_grad=True)
for call in (lambda: op.embedding(table, ids), lambda: op.distill_loss(logits, teacher, classes)):
    call()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    except RuntimeError as e:
        assert "native module" in str(e), e
    else:
        raise SystemExit("was not refused")
    with torch.cuda.graph(torch.cuda.CUDAGraph()), torch.no_grad():
        call()
print("refused")
"""


def test_a_captured_call_without_the_native_module():
    r = subprocess.run([sys.executable, "-c", WITHOUT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "refused" in r.stdout, r.stdout + r.stderr
