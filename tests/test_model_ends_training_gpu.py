"""A training step from tokens to weights: lookup in a table that the output layer shares, logits, the loss against a teacher, its
gradient, the table's gradient from both ends, and the optimizers of this package.

The allowances: u = 2^-24.  With |.| taken of every factor, a product over m terms is off by (m + 2) u of the same product of
absolute values, from which logits are off by e = (H + 2) u |h||w|.  An entry of dz moves by at most 2 a T e / T + 2 (1 - a) e
with the logits and is off by r of its terms itself (r as for the operator alone: under 600 u for 300 classes), so that dz is
off by  d = 2 e + 600 u size;  dW = dz^T h + S(dz W) is off by  d^T |h| + S(d |W|)  and by (N + V + H) u of its absolute
products.
"""
import pytest
import torch

from raf_b200 import distributed as dist
from raf_b200 import op, optim

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
N, V, H, K = 96, 301, 40, 8
HOW = dict(temperature=2.0, alpha=0.5, ignore_index=-100)
SCALE, LOSS_SCALE = H ** 0.5, 1024.0


def batch(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, H, generator=g, device="cuda") * 0.2
    tokens = torch.randint(0, V, (4, N // 4), generator=g, device="cuda")
    tokens[0, :5] = 7
    teacher = torch.randn(4, N // 4, K, generator=g, device="cuda")
    ids = torch.rand(N, V, generator=g, device="cuda").argsort(1)[:, :K].reshape(4, N // 4, K).contiguous()
    labels = torch.randint(0, V, (4, N // 4), generator=g, device="cuda")
    labels[1, ::3] = -100
    return w, tokens, teacher, ids, labels


def gradient_by_hand(w, tokens, teacher, ids, labels, weights):
    """The package's operators and plain matrix products, the gradient with the loss scale still in it."""
    h = op.embedding(w, tokens, SCALE)
    room = torch.zeros(N, V + 3, device="cuda")  # rows of logits further apart than they are long
    logits = room[:, :V]
    torch.mm(h.view(N, H), w.t(), out=logits)
    flat = [t.reshape((N,) + t.shape[2:]) for t in (teacher, ids, labels)]
    loss, dz = op.distill_loss_with_dpred(weights.reshape(N), logits, *flat, grad_scale=LOSS_SCALE, **HOW)
    dw = torch.mm(dz.t(), h.view(N, H))
    dh = torch.mm(dz, w)
    op.embedding_dx(dh.view(4, N // 4, H), tokens, V, SCALE, out=dw, accumulate=True)
    return loss.view(tokens.shape), dw


def gradient_in_64_bits(w, tokens, teacher, ids, labels, weights):
    x = w.double().requires_grad_()
    h = x[tokens].reshape(N, H) * SCALE
    z = h @ x.t()
    t, a = HOW["temperature"], HOW["alpha"]
    log_p = torch.log_softmax(teacher.double().reshape(N, K) / t, 1)
    log_q = torch.log_softmax(z / t, 1).gather(1, ids.reshape(N, K))
    y = labels.reshape(N)
    hard = -torch.log_softmax(z, 1).gather(1, y.clamp(min=0)[:, None])[:, 0]
    loss = (a * t * t * (log_p.exp() * (log_p - log_q)).sum(1) + (1 - a) * hard) * (y >= 0)
    (loss * weights.reshape(N).double()).sum().backward()
    with torch.no_grad():  # how far the result in fp32 may be off
        ah, aw, wt = h.abs(), w.double().abs(), weights.reshape(N, 1).double().abs() * (y >= 0)[:, None]
        e = ((H + 2) * U * (ah @ aw.t())).amax(1, keepdim=True)
        p = torch.zeros_like(z).scatter_add_(1, ids.reshape(N, K), log_p.exp())
        hot = torch.zeros_like(z).scatter_(1, y.clamp(min=0)[:, None], 1.0)
        size = (a * t * (torch.softmax(z / t, 1) + p) + (1 - a) * (torch.softmax(z, 1) + hot)) * wt
        d = 2 * e * wt + (600 + N + V + H) * U * size
        back = torch.zeros_like(x).index_add_(0, tokens.reshape(N), (d @ aw) * SCALE)
        allowed = d.t() @ ah + back
    return loss.detach().view(tokens.shape), x.grad, allowed


def test_a_step_of_a_tied_table():
    w, tokens, teacher, ids, labels = batch()
    weights = torch.rand(tokens.shape, device="cuda") / N
    loss, dw = gradient_by_hand(w, tokens, teacher, ids, labels, weights)
    want_loss, want, allowed = gradient_in_64_bits(w, tokens, teacher, ids, labels, weights)
    assert bool(((dw.double() / LOSS_SCALE - want).abs() <= allowed).all())
    assert bool((loss[labels < 0] == 0).all())
    assert float((loss.double() - want_loss).abs().max()) <= 2000 * U * (1 + float(want_loss.max()))

    # the same gradient by autograd, read from .grad by the optimizers
    p = torch.nn.Parameter(w.clone())
    z = op.embedding(p, tokens, SCALE) @ p.t()
    (op.distill_loss(z, teacher, ids, labels, **HOW)[0] * weights).sum().backward()
    assert bool(((p.grad.double() - want).abs() <= allowed).all())
    before = p.detach().clone()
    optim.SGD([p], 0.5, momentum=0.9).step()
    assert torch.equal(p.detach(), op.sgd(before, p.grad, torch.zeros_like(before), 0.5, 0.9)[1])

    # the optimizer takes the loss scale back
    x, v = w.clone(), torch.zeros_like(w)
    op.sgd_(x, dw, v, 0.5, 0.9, grad_scale=1 / LOSS_SCALE)
    assert bool(((x.double() - (w.double() - 0.5 * want)).abs() <= 0.5 * allowed + 4 * U * (w.double().abs() + want.abs())).all())
    lans = optim.LANS([p])
    lans.step()
    assert bool(p.isfinite().all()) and not torch.equal(p.detach(), x)


def test_micro_batches_into_the_gradient_of_a_zero_step():
    """Two micro-batches added up in the 16-bit gradient that with_sgd reads; the 16-bit table that it writes is looked up next."""
    g = torch.Generator(device="cuda").manual_seed(5)
    table = torch.randn(V, H, generator=g, device="cuda").bfloat16()
    wrapper = optim.with_sgd(learning_rate=1.0, momentum=0.0)({"table": table}, grad_dtype=torch.bfloat16)
    assert dist.get_communicator().size == 1
    grad = torch.empty_like(table)
    start, sums = table.double(), torch.zeros(V, H, dtype=torch.float64, device="cuda")
    absolute = torch.zeros_like(sums)
    for k in range(2):
        tokens = torch.randint(0, V, (N,), generator=g, device="cuda")
        dy = torch.randn(N, H, generator=g, device="cuda").bfloat16()
        op.embedding_dx(dy, tokens, V, SCALE, out=grad, accumulate=k > 0)
        sums.index_add_(0, tokens, dy.double() * SCALE)
        absolute.index_add_(0, tokens, dy.double().abs() * SCALE)
    # two roundings to bf16, of sums below `absolute`; fp32 in between
    allowed = absolute * (2 * 2.0 ** -8 * 1.01 + N * U)
    assert bool(((grad.double() - sums).abs() <= allowed).all())
    wrapper.step([grad])
    torch.cuda.synchronize()
    want = start - grad.double()
    assert bool(((table.double() - want).abs() <= want.abs() * 2.0 ** -8 + 2 * U * (start.abs() + grad.double().abs())).all())
    tokens = torch.arange(V, device="cuda").flip(0)
    assert torch.equal(op.embedding(table, tokens), table.flip(0))
    wrapper.close()


def test_a_captured_step():
    """Lookup, loss, both gradients and the update as one graph, replayed on new tokens."""
    w, tokens, teacher, ids, labels = batch(3)
    weights = torch.full(tokens.shape, 1.0 / N, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gradient_by_hand(w, tokens, teacher, ids, labels, weights)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dw = gradient_by_hand(w, tokens, teacher, ids, labels, weights)
    for seed in (4, 5):
        for old, new in zip((w, tokens, teacher, ids, labels), batch(seed)):
            old.copy_(new)
        graph.replay()
        want_loss, want, allowed = gradient_in_64_bits(w, tokens, teacher, ids, labels, weights)
        assert bool(((dw.double() / LOSS_SCALE - want).abs() <= allowed).all())
        assert float((loss.double() - want_loss).abs().max()) <= 2000 * U * (1 + float(want_loss.max()))
