"""The embedding and distillation operators through the native module and through ctypes: the same results, and what the module
hands back."""
import pytest
import torch

from raf_b200 import _lib, op

pytestmark = pytest.mark.gpu


def inputs(dtype=torch.bfloat16, n=37, v=130, h=24, k=5):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(v, h, generator=g, device="cuda").to(dtype)
    ids = torch.randint(-1, v + 1, (n,), generator=g, device="cuda")
    dy = torch.randn(n, h, generator=g, device="cuda").to(dtype)
    pred = torch.randn(n, v + 6, generator=g, device="cuda").to(dtype)[:, :v]
    teacher, classes = torch.randn(n, k, generator=g, device="cuda"), torch.randint(0, v, (n, k), generator=g, device="cuda")
    labels = torch.randint(-1, v, (n,), generator=g, device="cuda").int()
    return x, ids, dy, pred, teacher, classes, labels, torch.rand(n, generator=g, device="cuda")


def results():
    x, ids, dy, pred, teacher, classes, labels, w = inputs()
    into = torch.ones(130, 24, device="cuda")
    version = into._version
    op.embedding_dx(dy, ids, 130, 2.0, padding_idx=3, out=into, accumulate=True)
    assert into._version > version
    loss, stats = op.distill_loss(pred, teacher, classes, labels, 2.0, 0.5)
    both = op.distill_loss_with_dpred(w, pred, teacher, classes, labels, 3.0, 0.5, grad_scale=4.0)
    return [op.embedding(x, ids, 1.5), op.embedding(x, ids, dtype="float32"), op.embedding_dx(dy, ids, 130, dtype=torch.float32), into, loss, stats,
            op.distill_loss_dpred(torch.tensor(0.5, device="cuda"), pred, teacher, classes, stats, labels, 2.0, 0.5), *both,
            op.distill_loss(pred.contiguous(), teacher, classes)[0], op.distill_loss(pred[0], teacher[0], classes[0])[0]]


def test_both_ways_give_the_same(monkeypatch):
    want = results()
    monkeypatch.setattr(_lib, "_ops", _lib._GeneralWay())
    for a, b in zip(results(), want):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


def test_the_module_hands_back_what_is_unusual():
    x, ids, dy, pred, teacher, classes, labels, w = inputs()
    ops = _lib.ops()
    p = x.clone().requires_grad_()
    distill = lambda *a: ops.distill(None, *a[:3], None, a[3], 1.0, a[4], -100, 1.0, a[5])  # noqa: E731
    assert all(r is None for r in (
        ops.embedding(p, ids, 1.0, None), ops.embedding(x.cpu(), ids, 1.0, None), ops.embedding(x, ids.float(), 1.0, None), ops.embedding(x[0], ids, 1.0, None),
        ops.embedding(x.t(), ids, 1.0, None), ops.embedding(x.double(), ids, 1.0, None), ops.embedding(x, ids, "big", None), ops.embedding(x, ids, 1.0, "float32"),
        ops.embedding(x, ids, 1.0, torch.int8), ops.embedding_dx(dy, ids[:5], 130, 1.0, None, None, None, False), ops.embedding_dx(dy, ids, -1, 1.0, None, None, None, False),
        ops.embedding_dx(dy, ids, 1 << 31, 1.0, None, None, None, False), ops.embedding_dx(dy, ids, 130, 1.0, None, None, None, True),
        ops.embedding_dx(dy, ids, 37, 1.0, None, None, dy, False), ops.embedding_dx(dy, ids, 130, 1.0, None, None, x[:5], False),
        distill(pred, teacher, classes, None, 0.5, 0), distill(pred, teacher[:4], classes, None, 1.0, 0), distill(pred, teacher, classes, labels[:4], 1.0, 0),
        distill(pred.t(), teacher, classes, None, 1.0, 0), distill(pred, teacher, classes.float(), None, 1.0, 0), distill(pred, teacher, classes, None, 1.0, 1),
        distill(pred.detach().requires_grad_(), teacher, classes, None, 1.0, 0), distill(pred[:1].expand(37, 130), teacher, classes, None, 1.0, 0))), "a call went through"
    with torch.no_grad():
        assert torch.equal(ops.embedding(p, ids, 1.0, None), op.embedding(x, ids))
    with pytest.raises(_lib.RafB200Error):
        op.distill_loss(pred, teacher, classes, temperature=0.0)


def test_subclasses_and_modes_take_the_general_way():
    from torch.utils._python_dispatch import TorchDispatchMode

    x, ids = inputs()[:2]
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    with Mode():
        y = op.embedding(x, ids)
    assert seen and torch.equal(y, op.embedding(x, ids))


def test_out_of_memory_is_torchs_exception():
    x, ids = torch.zeros(10, 1 << 20, device="cuda"), torch.zeros(4000, dtype=torch.int64, device="cuda")
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (1 << 20)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            op.embedding(x, ids)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
