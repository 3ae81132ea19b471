"""The distillation loss and its gradient against the definition in 64 bits.

Where the allowances come from, with u = 2^-24 (half a step of fp32) and A the largest |z - max z| log2(e) / min(T, 1) of a
row that still matters (2^-126 is flushed to zero):
  an exponential    its argument is a rounded difference times a rounded constant, rounded: 3 A u in base 2, which is below 3 A u
                    relative; ex2.approx: 2 ulp = 4 u.  What is multiplied out of it (T = 2, 4) has its argument's error four
                    times at most with A a quarter, and 16 u + 3 u
  a sum             a thread of 128 or more keeps two sums of v / 256 terms at most, a lane of a short row sums of 32; they are merged
                    over 32 lanes, 8 warps, 8 blocks and rests: v / 256 + 64 additions, and a rescaling of 4 u with a batch of 32 terms
                    and with each merger
  a quotient        both of these, and a rounding
That is `r` below, relative, for q, r and the teacher's p: (v / 512 + 64) * 5 u covers the additions and the rescalings.  The
gradient is a difference of such terms, each off by r of itself, and is rounded once to the result's type.  A logarithm (2 ulp of
a value below log2(v) + A, which also bounds what is subtracted) is off by 4 u (A + log2 v) + r.
"""
import math
import os
import subprocess
import sys

import pytest
import torch

from raf_b200 import _lib, op

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
IGNORE = -100


def make(n, v, k, dtype, seed=0, pad=0, spread=2.0, index=torch.int64, labels=False, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + n * 31 + v * 7 + k)
    z = torch.randn(n, v, generator=g, device="cuda") * spread
    room = torch.full((n * (v + pad) + offset,), 77.0, dtype=dtype, device="cuda")
    pred = room[offset:].view(n, v + pad)[:, :v]
    pred.copy_(z)
    ids = torch.rand(n, v, generator=g, device="cuda").argsort(1)[:, :k].to(index).contiguous() if k <= v else torch.randint(0, v, (n, k), generator=g, device="cuda").to(index)
    teacher = (torch.randn(n, k, generator=g, device="cuda") * spread).to(dtype)
    lab = torch.randint(0, v, (n,), generator=g, device="cuda").to(index) if labels else None
    dy = torch.rand(n, generator=g, device="cuda") * 2 - 0.5
    return pred, teacher, ids, lab, dy


def definition(pred, teacher, ids, labels, temperature, alpha, ignore=IGNORE):
    """(loss, dz / 1, the sum of the absolute values of dz's terms, A)"""
    z, t, ids = pred.double(), teacher.double() / temperature, ids.long()
    n, v = z.shape
    here = (ids >= 0) & (ids < v)
    at = torch.where(here, ids, torch.zeros_like(ids))
    t = torch.where(here, t, torch.full_like(t, -math.inf))
    some = (t > -math.inf).any(1) | t.isnan().any(1)
    log_p = torch.log_softmax(t, 1)
    p = torch.where(some[:, None] & (log_p > -math.inf) | log_p.isnan() & some[:, None], log_p.exp(), torch.zeros_like(t))
    log_q, log_r = torch.log_softmax(z / temperature, 1), torch.log_softmax(z, 1)
    terms = torch.where(p == 0, torch.zeros_like(p), p * (log_p - log_q.gather(1, at)))
    weight = torch.zeros_like(z).scatter_add_(1, at, p)
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    grad, size = torch.zeros_like(z), torch.zeros_like(z)
    if alpha > 0:
        loss = loss + alpha * temperature ** 2 * terms.sum(1)
        q = torch.where(some[:, None], log_q.exp(), torch.zeros_like(z))
        grad = grad + alpha * temperature * (q - weight)
        size = size + alpha * temperature * (q + weight)
    if labels is not None:
        lab = labels.long()
        drop = (lab == ignore) | (lab < 0) | (lab >= v)
        hot = torch.zeros_like(z).scatter_(1, lab.clamp(0, v - 1)[:, None], 1.0)
        if alpha < 1:
            loss = loss - (1 - alpha) * log_r.gather(1, lab.clamp(0, v - 1)[:, None])[:, 0]
            grad = grad + (1 - alpha) * (log_r.exp() - hot)
            size = size + (1 - alpha) * (log_r.exp() + hot)
        loss = torch.where(drop, torch.zeros_like(loss), loss)
        grad = torch.where(drop[:, None], torch.zeros_like(grad), grad)
    span = (z.amax(1, keepdim=True) - torch.where(z > -math.inf, z, z.amax(1, keepdim=True))).nan_to_num(0, 0, 0).amax(1)
    return loss, grad, size, span * (math.log2(math.e) / min(temperature, 1.0))


def allowances(v, k, far, temperature, alpha):
    r = (4 + (v / 512 + 64) * 5 + k / 32 * 5 + 8) * U + 4 * far.clamp(max=126) * U
    # the loss: each of T^2's terms is a difference of logarithms
    loss = (alpha * temperature ** 2 + 1 - alpha) * ((far + math.log2(v) + 8) * 2 * r + 8 * U * (far + math.log2(v)))
    return r, loss


def check(args, loss=None, grad=None, dy=None, temperature=1.0, alpha=1.0, scale=1.0, ignore=IGNORE):
    pred, teacher, ids, labels = args
    want, g, size, far = definition(pred, teacher, ids, labels, temperature, alpha, ignore)
    t_far = (teacher.double().amax(1) - teacher.double().amin(1)).nan_to_num(0, 0, 0) / temperature * math.log2(math.e) if teacher.shape[1] else far * 0
    r, allowed = allowances(pred.shape[1], teacher.shape[1], torch.maximum(far, t_far), temperature, alpha)
    if loss is not None:
        same = (loss.double() == want) | (loss.isnan() & want.isnan())
        assert bool((same | ((loss.double() - want).abs() <= allowed)).all()), float(((loss.double() - want).abs() - allowed).max())
    if grad is not None:
        w = (torch.ones_like(want) if dy is None else dy.double() * torch.ones_like(want))[:, None] * scale
        g, size = g * w, size * w.abs()
        info = torch.finfo(grad.dtype)
        slack = size * (r[:, None] + 8 * U) + 2.0 ** -125 * w.abs()
        slack = slack + (g.abs() + slack) * info.eps / 2 + info.smallest_normal * info.eps / 2
        off = (grad.double() - g).abs()
        assert bool(((off <= slack) | (g.isnan() & grad.isnan())).all()), float((off - slack).max())


CASES = [(1, 1, 1), (2, 5, 3), (3, 17, 17), (1, 50257, 16), (40, 4096, 64), (300, 1000, 5), (7, 30522, 40), (5, 9001, 0), (160, 513, 100), (2, 131072, 33)]


@pytest.mark.parametrize("n,v,k", CASES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("temperature,alpha", [(1.0, 1.0), (2.0, 0.5), (0.7, 0.25), (1.0, 0.5), (3.0, 0.0), (4.0, 0.3)])
def test_loss_and_gradient(n, v, k, dtype, temperature, alpha):
    labels = alpha < 1
    pred, teacher, ids, lab, dy = make(n, v, k, dtype, index=torch.int32 if n % 2 else torch.int64, labels=labels, pad=0 if n % 3 else 7)
    if labels and n > 2:
        lab[1], lab[n // 2] = IGNORE, v
    if k > 2:
        ids[0, 1] = -1
        ids[-1, :] = v + 3  # no teacher at all
    how = dict(labels=lab, temperature=temperature, alpha=alpha)
    args = (pred, teacher, ids, lab)
    loss, stats = op.distill_loss(pred, teacher, ids, **how)
    assert loss.shape == (n,) and loss.dtype == F32
    check(args, loss, temperature=temperature, alpha=alpha)
    grad = op.distill_loss_dpred(dy, pred, teacher, ids, stats, grad_scale=64.0, **how)
    assert grad.shape == pred.shape and grad.dtype == dtype
    check(args, None, grad, dy, temperature, alpha, 64.0)
    both = op.distill_loss_with_dpred(dy, pred, teacher, ids, grad_scale=64.0, **how)
    check(args, both[0], both[1], dy, temperature, alpha, 64.0)
    again = op.distill_loss_with_dpred(dy, pred, teacher, ids, grad_scale=64.0, **how)
    assert torch.equal(both[0], again[0]) and torch.equal(both[1].view(torch.uint8), again[1].view(torch.uint8))


@pytest.mark.parametrize("v", list(range(1, 36)) + [511, 4095, 4097, 8193])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_length_at_every_address(v, dtype):
    for offset in range(0, 9, 1 if v < 20 else 3):
        args = make(5, v, min(v, 4), dtype, offset, pad=offset % 4, labels=True, offset=offset)
        pred, dy = args[0], args[4]
        room = torch.full((5 * (v + 3) + 5,), 9.0, dtype=dtype, device="cuda")
        out = room[5:].view(5, v + 3)[:, :v]
        how = dict(labels=args[3], temperature=2.0, alpha=0.5)
        loss, stats = op.distill_loss(pred, *args[1:3], **how)
        check(args[:4], loss, None, None, 2.0, 0.5)
        for call in (lambda o: op.distill_loss_dpred(dy, pred, *args[1:3], stats, out=o, **how),
                     lambda o: op.distill_loss_with_dpred(dy, pred, *args[1:3], out=o, **how)[1]):
            room.fill_(9.0)
            assert call(out) is out
            check(args[:4], None, out, dy, 2.0, 0.5)
            assert bool((room[:5] == 9).all()) and bool((room[5:].view(5, v + 3)[:, v:] == 9).all())
            check(args[:4], None, call(None), dy, 2.0, 0.5)


@pytest.mark.parametrize("n,v", [(3, 50257), (200, 1001), (2, 33)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_the_gradient_may_take_the_place_of_the_logits(n, v, dtype):
    pred, teacher, ids, lab, dy = make(n, v, 9, dtype, pad=5, labels=True)
    how = dict(labels=lab, temperature=1.5, alpha=0.3)
    stats = op.distill_loss(pred, teacher, ids, **how)[1]
    want = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
    alone = op.distill_loss_dpred(dy, pred, teacher, ids, stats, **how)
    for call, expect in ((lambda z: op.distill_loss_with_dpred(dy, z, teacher, ids, out=z, **how)[1], want[1]),
                         (lambda z: op.distill_loss_dpred(dy, z, teacher, ids, stats, out=z, **how), alone)):
        copy = torch.full((n, v + 5), 77.0, dtype=dtype, device="cuda")
        z = copy[:, :v]
        z.copy_(pred)
        assert call(z) is z
        check((pred, teacher, ids, lab), None, z, dy, 1.5, 0.3)
        assert bool((copy[:, v:] == 77).all())


def test_a_class_named_twice():
    pred, teacher, ids, lab, dy = make(6, 300, 8, F32, labels=True)
    ids[:, 3] = ids[:, 0]
    ids[1, :] = 5
    ids[2, 7] = ids[2, 0]
    lab[2] = ids[2, 0]
    lab[3] = ids[3, 5]
    for alpha in (1.0, 0.5):
        args = (pred, teacher, ids, lab)
        how = dict(labels=lab, temperature=2.0, alpha=alpha)
        loss, stats = op.distill_loss(*args[:3], **how)
        check(args, loss, op.distill_loss_dpred(dy, *args[:3], stats, **how), dy, 2.0, alpha)
        both = op.distill_loss_with_dpred(dy, *args[:3], **how)
        check(args, both[0], both[1], dy, 2.0, alpha)


@pytest.mark.parametrize("v", [2000, 9001, 40000])
@pytest.mark.parametrize("k", [1, 31, 33, 63, 64, 65, 1000, 1024])
def test_long_lists_of_entries(v, k):
    pred, teacher, ids, lab, dy = make(3, v, k, BF16)
    both = op.distill_loss_with_dpred(dy, pred, teacher, ids, temperature=2.0)
    check((pred, teacher, ids, None), both[0], both[1], dy, 2.0)
    stats = op.distill_loss(pred, teacher, ids, temperature=2.0)[1]
    check((pred, teacher, ids, None), None, op.distill_loss_dpred(dy, pred, teacher, ids, stats, temperature=2.0), dy, 2.0)
    ids.fill_(7)  # all of them one class
    both = op.distill_loss_with_dpred(dy, pred, teacher, ids, temperature=2.0)
    check((pred, teacher, ids, None), both[0], both[1], dy, 2.0)


def test_masked_logits():
    """Classes at -infinity or at the type's lowest value, in the student and in the teacher."""
    for dtype in (F32, F16, BF16):
        for low in (-math.inf, torch.finfo(dtype).min):
            pred, teacher, ids, lab, dy = make(6, 5003, 6, dtype, labels=True)
            pred[:, 100:4000] = low
            pred[1, :4990] = low
            ids[0], ids[1] = torch.arange(5, 11, device="cuda"), torch.arange(4990, 4996, device="cuda")
            ids[2:] = torch.randint(4000, 5003, ids[2:].shape, device="cuda")
            teacher[0, 2:] = -math.inf
            teacher[3] = -math.inf  # no teacher
            lab.copy_(torch.arange(4990, 4996, device="cuda"))
            for alpha, temperature in ((1.0, 2.0), (0.5, 2.0), (0.5, 1.0)):
                how = dict(labels=lab, temperature=temperature, alpha=alpha)
                both = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
                assert bool(both[1].isfinite().all()) and bool(both[0].isfinite().all())
                if low == -math.inf:
                    check((pred, teacher, ids, lab), both[0], both[1], dy, temperature, alpha)
                else:  # the lowest value is as good as -infinity: its exponential is 0
                    z = torch.where(pred == low, torch.full_like(pred, -math.inf), pred)
                    same = op.distill_loss_with_dpred(dy, z, teacher, ids, **how)
                    assert torch.equal(both[0], same[0]) and torch.equal(both[1], same[1])


def test_infinities_and_nan_stay_in_their_rows():
    pred, teacher, ids, lab, dy = make(9, 3001, 4, F32, labels=True)
    clean = op.distill_loss_with_dpred(dy, pred, teacher, ids, labels=lab, alpha=0.5)
    pred[1, 17] = math.nan
    pred[2, 3000] = math.inf
    pred[3] = -math.inf
    pred[4] = math.nan
    lab[4] = IGNORE  # a row that is left out may hold anything
    teacher[5, 1] = math.nan
    teacher[6, 0] = math.inf
    lab[7] = -5
    pred[8, ids[8, 0]] = -math.inf  # a class the teacher wants, and that cannot be
    loss, grad = op.distill_loss_with_dpred(dy, pred, teacher, ids, labels=lab, alpha=0.5)
    two = op.distill_loss(pred, teacher, ids, labels=lab, alpha=0.5)
    apart = op.distill_loss_dpred(dy, pred, teacher, ids, two[1], labels=lab, alpha=0.5)
    for x, d in ((loss, grad), (two[0], apart)):
        assert bool(x[[1, 2, 3, 5, 6]].isnan().all()) and bool((x[[4, 7]] == 0).all()) and float(x[8]) == math.inf
        assert bool((d[[4, 7]] == 0).all()) and bool(d[[1, 2, 3, 5, 6]].isnan().any(1).all()) and bool(d[8].isfinite().all())
        assert float(x[0]) == float(clean[0][0])
    assert torch.equal(grad[0], clean[1][0])


def test_a_term_without_weight_counts_nothing():
    pred, teacher, ids, lab, dy = make(4, 700, 5, F32, labels=True)
    pred[0, ids[0, 0]] = -math.inf
    pred[1, lab[1]] = -math.inf
    hard = op.distill_loss_with_dpred(dy, pred, teacher, ids, labels=lab, alpha=0.0, temperature=2.0)
    soft = op.distill_loss_with_dpred(dy, pred, teacher, ids, labels=lab, alpha=1.0, temperature=2.0)
    assert float(hard[0][1]) == math.inf and bool(hard[0][[0, 2, 3]].isfinite().all()) and bool(hard[1].isfinite().all())
    assert float(soft[0][0]) == math.inf and bool(soft[0][[1, 2, 3]].isfinite().all()) and bool(soft[1].isfinite().all())
    assert torch.equal(soft[1][2:], op.distill_loss_with_dpred(dy, pred, teacher, ids, temperature=2.0)[1][2:])


@pytest.mark.parametrize("n,v,dtype", [(3, 1000003, BF16), (2, 600001, F32), (310, 131073, F16), (200, 70001, F32)])
def test_rows_that_several_blocks_hold(n, v, dtype):
    """Few rows, and rows that are too long for the caches of a block each."""
    pred, teacher, _, lab, dy = make(n, v, 0, dtype, labels=True, pad=3)
    ids = torch.randint(0, v, (n, 5), device="cuda")
    teacher = torch.randn(n, 5, device="cuda")
    ids[:, 0], ids[:, 1] = 0, v - 1
    how = dict(labels=lab, temperature=2.0, alpha=0.5)
    both = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
    check((pred, teacher, ids, lab), both[0], both[1], dy, 2.0, 0.5)
    loss, stats = op.distill_loss(pred, teacher, ids, **how)
    check((pred, teacher, ids, lab), loss, op.distill_loss_dpred(dy, pred, teacher, ids, stats, **how), dy, 2.0, 0.5)


@pytest.mark.parametrize("v", [40, 3001, 30001])
def test_rows_of_one_value_alone(v):
    """A row of nothing but the type's lowest value, or of one other, says nothing: every class is as likely."""
    for dtype in (F32, F16, BF16):
        pred, teacher, ids, lab, dy = make(4, v, 3, dtype, labels=True)
        pred[0], pred[1], pred[2] = torch.finfo(dtype).min, torch.finfo(dtype).max, 0.0
        teacher[3, 1], ids[3, 1] = math.nan, -1  # what is absent may be anything
        for temperature, alpha in ((1.0, 0.5), (2.0, 0.5), (0.7, 0.5), (1.0, 1.0)):
            how = dict(labels=lab, temperature=temperature, alpha=alpha)
            both = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
            same = pred.clone()
            same[:3] = 0.0  # the definition of a constant row, without what 64 bits make of its subtractions
            t = teacher.clone()
            t[3, 1] = 0.0
            check((same, t, ids, lab), both[0], both[1], dy, temperature, alpha)


@pytest.mark.parametrize("shift", [0.0, 300.0, -3000.0])
def test_only_differences_of_logits_count(shift):
    """fp32 logits far from zero: their own spacing is 2^-12 at 3000, what is computed from them keeps fp32's steps."""
    pred, teacher, ids, lab, dy = make(8, 4000, 12, F32, labels=True)
    pred += shift
    teacher += shift
    for temperature, alpha in ((1.0, 0.5), (4.0, 0.5)):
        both = op.distill_loss_with_dpred(dy, pred, teacher, ids, labels=lab, temperature=temperature, alpha=alpha)
        check((pred, teacher, ids, lab), both[0], both[1], dy, temperature, alpha)


def test_more_than_32_bits_of_elements():
    n, v = 90000, 50257
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 60 GB")
    pred = torch.zeros(n, v, dtype=BF16, device="cuda")
    rows = torch.tensor([0, 85462, 89998, 89999], device="cuda")  # the 2^32nd element is in row 85461
    pred[rows] = torch.randn(4, v, device="cuda").to(BF16)
    teacher, ids = torch.randn(n, 5, device="cuda"), torch.randint(0, v, (n, 5), device="cuda")
    loss, stats = op.distill_loss(pred, teacher, ids, temperature=2.0)
    args = (pred[rows], teacher[rows], ids[rows], None)
    check(args, loss[rows], temperature=2.0)
    grad = op.distill_loss_dpred(None, pred, teacher, ids, stats, temperature=2.0)
    check(args, None, grad[rows], None, 2.0)
    check(args, op.distill_loss_with_dpred(None, pred, teacher, ids, temperature=2.0, out=grad)[0][rows], temperature=2.0)
    check(args, None, grad[rows], None, 2.0)


@pytest.mark.parametrize("v", [300, 9001])
def test_a_class_may_be_the_one_that_is_left_out(v):
    pred, teacher, ids, lab, dy = make(6, v, 4, BF16, labels=True, index=torch.int32)
    lab[1:4] = 0
    lab[4], lab[5] = -100, v + 7  # outside: left out as well
    how = dict(labels=lab, temperature=2.0, alpha=0.5, ignore_index=0)
    loss, stats = op.distill_loss(pred, teacher, ids, **how)
    check((pred, teacher, ids, lab), loss, op.distill_loss_dpred(dy, pred, teacher, ids, stats, **how), dy, 2.0, 0.5, ignore=0)
    both = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
    check((pred, teacher, ids, lab), both[0], both[1], dy, 2.0, 0.5, ignore=0)
    assert bool((both[0][1:] == 0).all()) and bool((both[1][1:] == 0).all()) and float(loss[0]) != 0


def test_weights_of_rows_and_shapes():
    pred, teacher, ids, lab, dy = make(12, 800, 4, F32, labels=True)
    how = dict(temperature=2.0, alpha=0.5)
    for lead in ((12,), (3, 4), (2, 1, 6)):
        z, t, i, y, w = pred.view(*lead, 800), teacher.view(*lead, 4), ids.view(*lead, 4), lab.view(lead), dy.view(lead)
        loss, stats = op.distill_loss(z, t, i, y, **how)
        assert loss.shape == lead and stats.shape == lead + (4,)
        grad = op.distill_loss_dpred(w, z, t, i, stats, y, **how)
        check((pred, teacher, ids, lab), loss.view(-1), grad.view(12, 800), dy, 2.0, 0.5)
    padded = torch.zeros(3, 4, 832, device="cuda")[..., :800]
    padded.copy_(pred.view(3, 4, 800))
    assert torch.equal(op.distill_loss(padded, teacher.view(3, 4, 4), ids.view(3, 4, 4), lab.view(3, 4), **how)[0].view(-1),
                       op.distill_loss(pred, teacher, ids, lab, **how)[0])
    one = torch.tensor(0.25, device="cuda")
    assert torch.equal(op.distill_loss_with_dpred(one, pred, teacher, ids)[1], op.distill_loss_with_dpred(None, pred, teacher, ids, grad_scale=0.25)[1])
    single = op.distill_loss(pred[0], teacher[0], ids[0])[0]
    assert single.shape == () and float(single) == float(op.distill_loss(pred[:1], teacher[:1], ids[:1])[0])
    empty = op.distill_loss_with_dpred(None, pred[:0], teacher[:0], ids[:0])
    assert empty[0].shape == (0,) and empty[1].shape == (0, 800)


def test_backward_is_dpred_and_the_slope():
    pred, teacher, ids, lab, dy = make(5, 600, 7, F32, labels=True)
    how = dict(labels=lab, temperature=2.0, alpha=0.4)
    z = pred.clone().requires_grad_()
    loss, stats = op.distill_loss(z, teacher, ids, **how)
    assert not stats.requires_grad
    (loss * dy).sum().backward()
    assert torch.equal(z.grad, op.distill_loss_dpred(dy, pred, teacher, ids, stats, **how))
    z.grad = None
    op.distill_loss(z, teacher, ids, **how)[0].mean().backward()  # a gradient that is broadcast
    mean = z.grad
    # differences of the loss, in fp32: steps of 2^-6, whose third order is 2^-12 of a second derivative below 4
    step = torch.zeros_like(pred)
    for j in (int(ids[2, 0]), int(lab[2]), 11):
        step.zero_()
        step[2, j] = 2.0 ** -6
        up, down = (op.distill_loss(pred + d, teacher, ids, **how)[0][2].double() for d in (step, -step))
        assert abs(float((up - down) * 32 / 5) - float(mean[2, j])) < 2e-4
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(op.distill_loss(z, teacher, ids)[0].sum(), z, create_graph=True)[0].sum(), z)


def test_streams_and_graphs():
    pred, teacher, ids, lab, dy = make(20, 3000, 7, BF16, labels=True)
    how = dict(labels=lab, temperature=2.0, alpha=0.4)
    want = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = op.distill_loss_with_dpred(dy, pred, teacher, ids, stream=side, **how)
    loss, stats = op.distill_loss(pred, teacher, ids, stream=side, **how)
    alone = op.distill_loss_dpred(dy, pred, teacher, ids, stats, stream=side, **how)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check((pred, teacher, ids, lab), loss, None, None, 2.0, 0.4)
    check((pred, teacher, ids, lab), None, alone, dy, 2.0, 0.4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
    pred.copy_(torch.randn(pred.shape, device="cuda"))
    graph.replay()
    check((pred, teacher, ids, lab), captured[0], captured[1], dy, 2.0, 0.4)


def test_refusals_on_the_gpu():
    pred, teacher, ids, lab, dy = make(6, 40, 3, F32, labels=True)
    stats = op.distill_loss(pred, teacher, ids)[1]
    big = torch.zeros(6, 2000, 1025, device="cuda")[0]
    bad = [lambda: op.distill_loss(pred.t(), teacher, ids), lambda: op.distill_loss(pred, teacher[:5], ids), lambda: op.distill_loss(pred, teacher, ids[:, :2]),
           lambda: op.distill_loss(pred, teacher, ids, alpha=0.5), lambda: op.distill_loss(pred, teacher, ids, lab[:5], alpha=0.5),
           lambda: op.distill_loss(pred, teacher, ids.cpu()), lambda: op.distill_loss(pred.expand(6, 6, 40), teacher, ids),
           lambda: op.distill_loss(pred[:1].expand(6, 40), teacher, ids), lambda: op.distill_loss(pred[:, :0], teacher, ids),
           lambda: op.distill_loss(pred, teacher.clone().requires_grad_(), ids),
           lambda: op.distill_loss_dpred(dy[:4], pred, teacher, ids, stats), lambda: op.distill_loss_dpred(dy, pred, teacher, ids, stats[:5]),
           lambda: op.distill_loss_dpred(dy, pred, teacher, ids, stats, out=pred.half()), lambda: op.distill_loss_dpred(dy, pred, teacher, ids, stats, out=pred[:5]),
           lambda: op.distill_loss_with_dpred(dy, pred, teacher, ids, out=torch.zeros(40, 6, device="cuda").t())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: op.distill_loss(pred.double(), teacher, ids), lambda: op.distill_loss(pred, teacher, ids.float()),
                 lambda: op.distill_loss(pred, teacher.double(), ids), lambda: op.distill_loss_dpred(dy.half(), pred, teacher, ids, stats)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: op.distill_loss(pred, teacher, ids, temperature=0.0), lambda: op.distill_loss(pred, teacher, ids, temperature=math.nan),
                 lambda: op.distill_loss(pred, teacher, ids, lab, alpha=1.5), lambda: op.distill_loss(big, big, torch.zeros(2000, 1025, dtype=torch.int32, device="cuda"))):
        with pytest.raises(_lib.RafB200Error):
            call()
    room = torch.zeros(6, 80, device="cuda")
    with pytest.raises(_lib.RafB200Error, match="overlaps"):
        op.distill_loss_with_dpred(dy, room[:, :40], teacher, ids, out=room[:, 40:])


@pytest.mark.parametrize("v", [300, 9001, 50257])
def test_statistics_from_elsewhere(v):
    """Maximum and sums by another program, nothing in the fourth place: whether a row has a teacher is read from its list."""
    for labels, temperature in ((False, 2.0), (True, 2.0), (False, 1.0)):
        pred, teacher, ids, lab, dy = make(7, v, 2, BF16, labels=labels)
        ids[2:5] = -1
        ids[5, 0] = v
        z = pred.double()
        top = z.amax(1, keepdim=True)
        stats = torch.stack([top[:, 0], ((z - top) / temperature).exp().sum(1), (z - top).exp().sum(1), torch.zeros_like(dy)], 1).float()
        how = dict(labels=lab, temperature=temperature, alpha=0.5 if labels else 1.0)
        for into in (None, pred.clone()):
            z = pred if into is None else into
            check((pred, teacher, ids, lab), None, op.distill_loss_dpred(dy, z, teacher, ids, stats, out=into, **how), dy, temperature, how["alpha"])


@pytest.mark.parametrize("v", [300, 9001, 40000])
def test_a_teacher_without_weight_may_hold_anything(v):
    """alpha = 0: neither loss nor gradient looks at the teacher's logits."""
    pred, teacher, ids, lab, dy = make(5, v, 5, BF16, labels=True)
    wild = teacher.clone()
    wild[0, 1], wild[1], wild[2, 0], wild[3] = math.nan, math.nan, math.inf, -math.inf
    for temperature in (1.0, 2.0, 3.0, 4.0):
        how = dict(labels=lab, temperature=temperature, alpha=0.0)
        loss, stats = op.distill_loss(pred, wild, ids, **how)
        check((pred, teacher, ids, lab), loss, op.distill_loss_dpred(dy, pred, wild, ids, stats, **how), dy, temperature, 0.0)
        both = op.distill_loss_with_dpred(dy, pred, wild, ids, **how)
        check((pred, teacher, ids, lab), both[0], both[1], dy, temperature, 0.0)


@pytest.mark.parametrize("v", [300, 9001, 40000])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_a_row_without_any_term_says_nothing(v, temperature):
    """No teacher, and no labels or no weight for them: loss and gradient 0, for a row of nothing but -infinity too."""
    pred, teacher, ids, lab, dy = make(5, v, 5, F16, labels=True)
    pred[:2] = -math.inf
    ids[0], ids[2], teacher[1] = -1, v, -math.inf
    for labels in (None, lab):
        how = dict(labels=labels, temperature=temperature, alpha=1.0)
        loss, stats = op.distill_loss(pred, teacher, ids, **how)
        both = op.distill_loss_with_dpred(dy, pred, teacher, ids, **how)
        for x, d in ((loss, op.distill_loss_dpred(dy, pred, teacher, ids, stats, **how)), both):
            assert bool((x[:3] == 0).all()) and bool((d[:3] == 0).all())
            check((pred[3:], teacher[3:], ids[3:], None if labels is None else lab[3:]), x[3:], d[3:], dy[3:], temperature)


@pytest.mark.parametrize("v", [300, 9001, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_the_statistics_hold(v, dtype):
    """A row's maximum, its sum at the temperature and its sum at one; NaN in place of what the loss does not sum up, and so is a
    gradient that takes it."""
    pred, teacher, ids, lab, dy = make(6, v, 3, dtype, labels=True)
    z = pred.double()
    top = z.amax(1)
    sums = [((z - top[:, None]) / t).exp().sum(1) for t in (1.0, 2.0)]
    for labels, temperature, alpha in ((None, 1.0, 1.0), (None, 2.0, 1.0), (lab, 1.0, 1.0), (lab, 2.0, 1.0), (lab, 1.0, 0.5), (lab, 2.0, 0.5), (lab, 2.0, 0.0)):
        stats = op.distill_loss(pred, teacher, ids, labels, temperature, alpha)[1]
        r, _ = allowances(v, 0, definition(pred, teacher, ids, None, 1.0, 1.0)[3], 1.0, 1.0)
        assert torch.equal(stats[:, 0].double(), top)
        assert bool(((stats[:, 1].double() - sums[int(temperature) - 1]).abs() <= r * sums[int(temperature) - 1]).all())
        if temperature == 1.0 or alpha < 1:
            assert bool(((stats[:, 2].double() - sums[0]).abs() <= r * sums[0]).all())
        else:
            assert bool(stats[:, 2].isnan().all())
            assert bool(op.distill_loss_dpred(dy, pred, teacher, ids, stats, lab, temperature, 0.5).isnan().all())
    lab[2], lab[4] = IGNORE, v
    stats = op.distill_loss(pred, teacher, ids, lab, 2.0, 0.5)[1]
    left_out = torch.tensor([False, False, True, False, True, False], device="cuda")
    assert torch.equal(stats[:, :3].isnan().all(1), left_out) and torch.equal(stats[:, :3].isnan().any(1), left_out)
    assert torch.equal(op.distill_loss_dpred(dy, pred, teacher, ids, stats, temperature=2.0).isnan().all(1), left_out)
    assert bool((op.distill_loss_dpred(dy, pred, teacher, ids, stats, lab, 2.0, 0.5)[left_out] == 0).all())


def test_forward_mode_and_lazy_signs_are_refused():
    """Tensors whose tangent, or whose sign, is not at their address."""
    import torch.autograd.forward_ad as fwd

    pred, teacher, ids, lab, dy = make(6, 40, 3, F32, labels=True)
    stats = op.distill_loss(pred, teacher, ids)[1]

    def calls(z, t, w):
        plain = z is pred and t is teacher
        return ([] if plain else [lambda: op.distill_loss(z, t, ids), lambda: op.distill_loss(z, t, ids, stream=torch.cuda.current_stream())]) + [
            lambda: op.distill_loss_dpred(w, z, t, ids, stats), lambda: op.distill_loss_with_dpred(w, z, t, ids),
            lambda: op.distill_loss_dpred(w, z, t, ids, stats, out=torch.empty_like(pred))]

    with fwd.dual_level():
        z, t, w = (fwd.make_dual(x, torch.ones_like(x)) for x in (pred, teacher, dy))
        for call in calls(z, teacher, dy) + calls(pred, t, dy) + calls(pred, teacher, w):
            with pytest.raises(ValueError, match="forward"):
                call()
        with torch.no_grad(), pytest.raises(ValueError, match="forward"):
            op.distill_loss(z, teacher, ids)
        with pytest.raises(ValueError, match="forward"):
            op.distill_loss(fwd.make_dual(pred.clone().requires_grad_(), torch.ones_like(pred)), teacher, ids)
        assert torch.equal(op.distill_loss(pred, teacher, ids)[1], stats)
    for call in calls(torch._neg_view(pred), teacher, dy) + calls(pred, torch._neg_view(teacher), dy) + calls(pred, teacher, torch._neg_view(dy)):
        with pytest.raises(ValueError, match="negat"):
            call()


def test_a_gradient_is_not_written_into_a_graph():
    """out takes data: it requires no gradient itself, unless it is pred, whose graph ends there."""
    pred, teacher, ids, lab, dy = make(6, 40, 3, F32, labels=True)
    stats = op.distill_loss(pred, teacher, ids)[1]
    out = torch.zeros_like(pred).requires_grad_()
    for call in (lambda: op.distill_loss_dpred(dy, pred, teacher, ids, stats, out=out), lambda: op.distill_loss_with_dpred(dy, pred, teacher, ids, out=out * 2)):
        with pytest.raises(ValueError, match="gradient"):
            call()
    want = op.distill_loss_dpred(dy, pred, teacher, ids, stats)
    with torch.no_grad():
        assert torch.equal(op.distill_loss_dpred(dy, pred, teacher, ids, stats, out=out), want)
    w = pred.clone().requires_grad_()
    logits = w * 1.0
    op.distill_loss_dpred(dy, logits, teacher, ids, stats, out=logits)
    assert torch.equal(logits, want)


ALONE = """
import sys
sys.path.insert(0, {tests!r})
from test_distill_gpu import *

"""


def alone(body):
    """Runs `body` in a process of its own, where no call has gone before."""
    script = ALONE.format(tests=os.path.dirname(os.path.abspath(__file__))) + body + "\nprint('went through')\n"
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "went through" in r.stdout, r.stdout + r.stderr


def test_lists_whose_entries_just_fill_the_shared_memory_that_is_given_unasked():
    """48 KB for what a block asks for and what its kernel declares together: from 32 KB for the logits and 754 entries on that is
    more, before the entries alone are."""
    alone("""
for k in (752, 753, 754, 760, 767, 768):
    pred, teacher, ids, lab, dy = make(3, 40000, k, BF16)
    loss, stats = op.distill_loss(pred, teacher, ids)
    both = op.distill_loss_with_dpred(dy, pred, teacher, ids)
    check((pred, teacher, ids, None), loss, op.distill_loss_dpred(dy, pred, teacher, ids, stats), dy)
    check((pred, teacher, ids, None), both[0], both[1], dy)
""")


def test_first_calls_of_several_threads():
    """Lists of two lengths above 48 KB, the first of their kernel, at the same time; and the longer one again."""
    alone("""
import threading

failed = []
for dtype in (F32, F16, BF16):
    pred, teacher, ids, lab, dy = make(3, 300, 1000, dtype, labels=True)
    stats = torch.ones(3, 4, device="cuda")
    lists = [(teacher[:, :600].contiguous(), ids[:, :600].contiguous()), (teacher, ids)]
    for how in (dict(), dict(labels=lab, alpha=0.5, temperature=2.0), dict(labels=lab, alpha=0.5, temperature=4.0), dict(labels=lab, alpha=0.5, temperature=3.0)):
        for call in (lambda t, i: op.distill_loss(pred, t, i, **how), lambda t, i: op.distill_loss_with_dpred(dy, pred, t, i, **how),
                     lambda t, i: op.distill_loss_dpred(dy, pred, t, i, stats, **how)):
            start = threading.Barrier(4)

            def first(*args):
                start.wait()
                try:
                    call(*args)
                except Exception as e:
                    failed.append(repr(e))

            threads = [threading.Thread(target=first, args=args) for args in lists * 2]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            call(*lists[1])
torch.cuda.synchronize()
assert not failed, failed
""")
