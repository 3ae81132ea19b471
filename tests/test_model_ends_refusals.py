"""What the embedding and distillation operators refuse before any launch: CPU tensors, and bad arguments of the C ABI."""
import ctypes as C

import pytest
import torch

from raf_b200 import _lib, op

AT = 1 << 20  # an address that nothing looks at


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    dy, pred, teacher, classes = torch.zeros(3, 8), torch.zeros(3, 9), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: op.embedding(x, ids), lambda: op.embedding_dx(dy, ids, 4), lambda: op.distill_loss(pred, teacher, classes),
                 lambda: op.distill_loss_dpred(None, pred, teacher, classes, torch.zeros(3, 4)),
                 lambda: op.distill_loss_with_dpred(None, pred, teacher, classes)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_embedding_arguments():
    lib = _lib.load()

    def call(x=AT, dtype=_lib.F32, rows=4, width=8, ids=AT, index=_lib.I64, n=3, out=AT, out_dtype=_lib.F32):
        return lib.rafb200_embedding(x, dtype, rows, width, ids, index, n, 1.0, out, out_dtype, None)

    for bad in (dict(dtype=3), dict(out_dtype=9), dict(index=_lib.F32), dict(index=5), dict(rows=-1), dict(width=-1), dict(n=-1), dict(x=None),
                dict(ids=None), dict(out=None), dict(n=1 << 60, width=1 << 10), dict(rows=1 << 60, width=1 << 10), dict(n=1 << 50)):
        assert call(**bad) == 1, bad
    assert call(n=0, x=None, ids=None, out=None) == 0 and call(width=0, x=None, ids=None, out=None) == 0


def test_embedding_dx_arguments():
    lib = _lib.load()

    def call(dy=AT, dtype=_lib.F32, ids=AT, index=_lib.I32, n=3, rows=4, width=8, accumulate=0, dx=AT, dx_dtype=_lib.F32, ws=AT, ws_bytes=1 << 20):
        return lib.rafb200_embedding_dx(dy, dtype, ids, index, n, rows, width, 1.0, -1, accumulate, dx, dx_dtype, ws, ws_bytes, None)

    need = lib.rafb200_embedding_dx_workspace_bytes(3, 8)
    assert need > 0
    for bad in (dict(dtype=3), dict(dx_dtype=-1), dict(index=_lib.F32), dict(n=-1), dict(rows=-1), dict(width=-1), dict(n=1 << 31, ws_bytes=1 << 60),
                dict(rows=1 << 31), dict(dy=None), dict(ids=None), dict(dx=None), dict(ws=None), dict(ws_bytes=need - 1), dict(ws=AT + 4)):
        assert call(**bad) == 1, bad
    assert call(rows=0, dx=None) == 0 and call(width=0, dx=None) == 0 and call(n=0, accumulate=1, dx=None, ws=None) == 0
    assert lib.rafb200_embedding_dx_workspace_bytes(0, 8) == 0 and lib.rafb200_embedding_dx_workspace_bytes(-1, 8) == 0


def test_distill_arguments():
    lib = _lib.load()
    good = dict(pred=AT, teacher_logits=AT, teacher_ids=AT, labels=AT, n=2, v=10, ld=10, ignore_index=-100, temperature=2.0, alpha=0.5, k=3,
                pred_dtype=_lib.F32, teacher_dtype=_lib.F32, ids_dtype=_lib.I64, labels_dtype=_lib.I32)

    def calls(dy=AT, out=2 * AT, ld_out=10, stats=AT, loss=AT, **changed):
        d = _lib.Distill(**dict(good, **changed))
        return (lib.rafb200_distill_loss(C.byref(d), loss, stats, None), lib.rafb200_distill_loss_dpred(C.byref(d), dy, 1, 1.0, stats, out, ld_out, None),
                lib.rafb200_distill_loss_with_dpred(C.byref(d), dy, 1, 1.0, loss, out, ld_out, None))

    nan, inf = float("nan"), float("inf")
    for bad in (dict(pred_dtype=3), dict(teacher_dtype=-1), dict(ids_dtype=0), dict(labels_dtype=2), dict(n=-1), dict(n=1 << 28), dict(v=0), dict(v=1 << 31),
                dict(k=-1), dict(k=1025), dict(ld=9), dict(ld=1 << 32), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=nan), dict(temperature=inf),
                dict(temperature=1e-30), dict(alpha=-0.1), dict(alpha=1.1), dict(alpha=nan), dict(labels=None), dict(pred=None), dict(teacher_logits=None), dict(teacher_ids=None)):
        assert calls(**bad) == (1, 1, 1), bad
    assert calls(n=0, pred=None, teacher_logits=None, teacher_ids=None, out=None, stats=None, loss=None) == (0, 0, 0)
    assert calls(loss=None, stats=None, out=None) == (1, 1, 1)
    assert calls(stats=AT + 4, ld_out=9) == (1, 1, 1)
    assert calls(out=AT + 4, stats=None) == (1, 1, 1)  # the gradient begins inside pred
    assert calls(out=AT - 4, stats=None) == (1, 1, 1)  # and ends inside it
    assert calls(out=AT, ld_out=11, stats=None) == (1, 1, 1)  # at pred's address, with other rows
    assert lib.rafb200_distill_loss(None, AT, AT, None) == 1


def test_without_the_native_module_no_captured_graph(monkeypatch):
    """Whether a captured backward would end the process the native module alone can say."""
    x = torch.zeros(3, requires_grad=True)
    monkeypatch.setattr(_lib, "_ops", _lib._GeneralWay())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="native module"):
        op._check_capturable("embedding", x)
