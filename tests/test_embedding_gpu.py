"""raf.op.embedding and raf.op.embedding_dx against the definition in 64 bits.

A lookup is one product in fp32 (off by half a step of fp32) and one rounding.  A sum of m terms in fp32, in
whatever order, is off by at most m half steps of the sum of the absolute values (the products with the scale and
the addition to what is there: two more); then comes the rounding to the result's type, half a step of the value
or, below the smallest normal number, half the smallest subnormal one.
"""
import pytest
import torch

from raf_b200 import _lib, op

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype, value):
    return value.abs() * half_step(dtype) + torch.finfo(dtype).smallest_normal * half_step(dtype)


def ids_of(kind, n, rows, g, dtype=torch.int64):
    if kind == "uniform":
        t = torch.randint(0, rows, (n,), generator=g, device="cuda")
    elif kind == "one":
        t = torch.full((n,), rows - 1, device="cuda")
    elif kind == "falling":
        t = (torch.arange(n, device="cuda") % rows).flip(0)
    elif kind == "words":  # a few very often
        t = ((torch.rand(n, generator=g, device="cuda") ** 6) * rows).long().clamp_(max=rows - 1)
    else:  # outside on both sides, the largest and smallest numbers among them
        t = torch.randint(-2, rows + 3, (n,), generator=g, device="cuda")
        if n > 4:
            info = torch.iinfo(dtype)
            t[0], t[2] = info.max, info.min
    return t.to(dtype)


def lookup_of(x, ids, scale):
    ids = ids.long()
    inside = (ids >= 0) & (ids < x.shape[0])
    rows = x.double()[ids.clamp(0, max(x.shape[0] - 1, 0))] if x.shape[0] else torch.zeros(ids.shape + x.shape[1:], device="cuda", dtype=torch.float64)
    return torch.where(inside[..., None], rows * scale, torch.zeros_like(rows))


def gradient_of(dy, ids, rows, scale, padding=-1):
    ids = ids.long()
    counted = (ids >= 0) & (ids < rows) & (ids != padding)
    to = torch.where(counted, ids, torch.full_like(ids, rows)).reshape(-1)
    d = dy.double().reshape(-1, dy.shape[-1])
    zero = torch.zeros(rows + 1, dy.shape[-1], dtype=torch.float64, device="cuda")
    count = torch.zeros(rows + 1, dtype=torch.float64, device="cuda").index_add_(0, to, torch.ones_like(to, dtype=torch.float64))
    return zero.index_add(0, to, d)[:-1] * scale, zero.index_add(0, to, d.abs())[:-1] * abs(scale), count[:-1, None]


def check_gradient(got, dy, ids, rows, scale, padding=-1, before=None):
    want, size, count = gradient_of(dy, ids, rows, scale, padding)
    if before is not None:
        want, size = want + before.double(), size + before.double().abs()
    off = (got.double() - want).abs()
    allowed = (count + 2) * HALF32 * size * (1 + 2 ** -10)
    allowed += rounding(got.dtype, want.abs() + allowed)
    assert bool((off <= allowed).all()), float((off - allowed).max())
    if before is not None:  # rows without a token are not touched
        quiet = (count == 0)[:, 0]
        assert torch.equal(got[quiet].view(torch.uint8), before[quiet].view(torch.uint8))


@pytest.mark.parametrize("n,rows,width", [(0, 5, 8), (1, 1, 1), (3, 7, 2), (5, 4, 0), (33, 1000, 136), (129, 513, 1023), (1000, 31, 1024),
                                          (64, 9, 4097), (2049, 30522, 24)])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (F32, BF16), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F16)])
def test_lookup(n, rows, width, dtype, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(n + rows + width)
    x = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    for kind, index, scale in (("uniform", torch.int64, 1.0), ("outside", torch.int32, 31.984)):
        ids = ids_of(kind, n, rows, g, index)
        got = op.embedding(x, ids, scale, dtype=out_dtype)
        want = lookup_of(x, ids, scale)
        assert got.shape == want.shape and got.dtype == out_dtype
        if dtype == out_dtype and scale == 1.0:
            assert torch.equal(got.double(), want)
        slack = want.abs() * 2 * HALF32  # of the scale and of the product
        assert bool(((got.double() - want).abs() <= slack + rounding(out_dtype, want.abs() + slack)).all())


@pytest.mark.parametrize("width", [255, 256, 257, 300, 1022, 1029])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (F32, BF16), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F16)])
def test_wide_rows_at_any_address(width, dtype, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(width)
    n, rows = 57, 30
    ids = ids_of("outside", n, rows, g)
    for a, b in ((0, 0), (1, 0), (0, 1), (3, 2), (7, 5)):
        x = torch.randn(rows * width + a, generator=g, device="cuda").to(dtype)[a:].view(rows, width)
        room = torch.full((n * width + b + 9,), 7.0, dtype=out_dtype, device="cuda")
        out = room[b:b + n * width].view(n, width)
        op.embedding(x, ids, 0.75, dtype=out_dtype, out=out)
        want = lookup_of(x, ids, 0.75)
        slack = want.abs() * HALF32
        assert bool(((out.double() - want).abs() <= slack + rounding(out_dtype, want.abs() + slack)).all())
        assert bool((room[:b] == 7).all()) and bool((room[b + n * width:] == 7).all())


@pytest.mark.parametrize("shift", [1, 2, 4])
def test_tables_and_results_at_any_address(shift):
    g = torch.Generator(device="cuda").manual_seed(shift)
    ids = ids_of("words", 300, 50, g)
    for dtype in (F32, BF16):
        flat = torch.randn(50 * 40 + shift, generator=g, device="cuda").to(dtype)
        x = flat[shift:].view(50, 40)
        out = torch.empty(300 * 40 + 3 * shift, dtype=dtype, device="cuda").fill_(7)
        op.embedding(x, ids, out=out[shift:shift + 300 * 40].view(300, 40))
        assert torch.equal(out[shift:shift + 300 * 40].view(300, 40), x[ids])
        assert bool((out[:shift] == 7).all()) and bool((out[shift + 300 * 40:] == 7).all())
        dy = torch.randn(300 * 40 + shift, generator=g, device="cuda").to(dtype)[shift:].view(300, 40)
        room = torch.empty(50 * 40 + 3 * shift, dtype=dtype, device="cuda").fill_(7)
        dx = room[shift:shift + 50 * 40].view(50, 40)
        op.embedding_dx(dy, ids, 50, 0.5, out=dx)
        check_gradient(dx, dy, ids, 50, 0.5)
        assert bool((room[:shift] == 7).all()) and bool((room[shift + 50 * 40:] == 7).all())


def test_shapes_of_indices():
    x = torch.randn(11, 6, device="cuda")
    for shape in ((), (3,), (2, 5), (2, 0, 4), (2, 1, 3)):
        ids = torch.randint(0, 11, shape, device="cuda")
        assert torch.equal(op.embedding(x, ids), x[ids])
        dx = op.embedding_dx(torch.ones(shape + (6,), device="cuda"), ids, 11)
        assert torch.equal(dx[:, 0], torch.bincount(ids.reshape(-1), minlength=11).float())


@pytest.mark.parametrize("n,rows,width", [(0, 5, 8), (1, 1, 1), (1, 3, 1024), (7, 2, 3), (31, 513, 64), (257, 2, 1024), (1000, 40, 1023), (3000, 512, 136),
                                          (20011, 30522, 40), (9000, 2, 264), (4097, 300000, 8), (70001, 1000, 18), (12, 4, 5000), (300007, 5000, 6), (140001, 2, 33)])
@pytest.mark.parametrize("kind", ["uniform", "one", "falling", "words", "outside"])
def test_gradient(n, rows, width, kind):
    g = torch.Generator(device="cuda").manual_seed(n + 3 * rows + width)
    for dtype, out_dtype, index, scale, padding in ((BF16, BF16, torch.int64, 1.0, -1), (F32, F32, torch.int32, 22.627, 0), (F16, F32, torch.int64, 0.25, rows - 1)):
        ids = ids_of(kind, n, rows, g, index)
        dy = torch.randn(n, width, generator=g, device="cuda").to(dtype)
        got = op.embedding_dx(dy, ids, rows, scale, padding_idx=padding, dtype=out_dtype)
        assert got.shape == (rows, width) and got.dtype == out_dtype
        check_gradient(got, dy, ids, rows, scale, padding)
        again = op.embedding_dx(dy, ids, rows, scale, padding_idx=padding, dtype=out_dtype)
        assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))
        before = torch.randn(rows, width, generator=g, device="cuda").to(out_dtype)
        into = before.clone()
        assert op.embedding_dx(dy, ids, rows, scale, padding_idx=padding, out=into, accumulate=True) is into
        check_gradient(into, dy, ids, rows, scale, padding, before)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 511, 512, 513, 262143, 262144, 262145])
def test_every_digit_of_an_id_counts(rows):
    """Tables at the borders of the sort's digits: one token for the first and the last rows."""
    ids = torch.tensor([rows - 1, 0, rows // 2, rows - 1, rows, -1], device="cuda")
    dy = torch.arange(1, 7, device="cuda", dtype=F32)[:, None].expand(6, 3).contiguous()
    got = op.embedding_dx(dy, ids, rows)
    check_gradient(got, dy, ids, rows, 1.0)


def test_infinities_and_nan_stay_in_their_rows():
    ids = torch.tensor([3, 1, 3, 2, 9], device="cuda")
    dy = torch.ones(5, 16, device="cuda")
    dy[1], dy[2], dy[4] = float("nan"), float("inf"), float("nan")  # index 9 names no row
    got = op.embedding_dx(dy, ids, 5)
    assert bool(got[1].isnan().all()) and bool((got[3] == float("inf")).all())
    assert bool((got[[0, 4]] == 0).all()) and bool((got[2] == 1).all())
    into = torch.full((5, 16), 2.0, device="cuda")
    op.embedding_dx(dy, ids, 5, out=into, accumulate=True)
    assert bool((into[[0, 4]] == 2).all()) and bool((into[2] == 3).all())


def test_more_than_32_bits_of_elements():
    width, n, rows = 65536, 65600, 65700  # 4.3e9 elements each
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.empty(rows, width, dtype=BF16, device="cuda")
    x[-1], x[65535], x[0] = 3, 5, 7
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    ids[-1], ids[-2] = rows - 1, 65535
    y = op.embedding(x, ids)
    assert bool((y[-1] == 3).all()) and bool((y[-2] == 5).all()) and bool((y[:2] == 7).all())
    del x
    y.zero_()
    y[-1], y[-2], y[3] = 1, 2, 4
    dx = op.embedding_dx(y, ids, rows)
    assert bool((dx[-1] == 1).all()) and bool((dx[65535] == 2).all()) and bool((dx[0] == 4).all())
    assert int(torch.count_nonzero(dx)) == 3 * width


def test_on_another_stream_and_in_a_graph():
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = torch.randn(700, 96, generator=g, device="cuda"), torch.randn(5000, 96, generator=g, device="cuda")
    ids = ids_of("words", 5000, 700, g)
    want = op.embedding_dx(dy, ids, 700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y, dx = op.embedding(x, ids, stream=side), op.embedding_dx(dy, ids, 700, stream=side)
    side.synchronize()
    assert torch.equal(y, x[ids]) and torch.equal(dx, want)
    # two graphs, each with a workspace of its own, replayed at the same time with new data
    graphs, outs, inputs = [], [], [(dy.clone(), ids.clone()) for _ in range(2)]
    for d, i in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(op.embedding_dx(d, i, 700))
        graphs.append(graph)
    for k, (d, i) in enumerate(inputs):
        d.copy_(torch.randn(d.shape, generator=g, device="cuda"))
        i.copy_(ids_of("words", 5000, 700, g))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for s, graph in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for (d, i), got in zip(inputs, outs):
        assert torch.equal(got, op.embedding_dx(d, i, 700))


def test_backward_is_embedding_dx():
    x = torch.randn(50, 24, device="cuda", requires_grad=True)
    ids = torch.randint(0, 50, (4, 9), device="cuda")
    y = op.embedding(x, ids, 3.0, padding_idx=2)
    assert torch.equal(y.detach(), x.detach()[ids] * 3.0)
    w = torch.randn(4, 9, 24, device="cuda")
    (y * w).sum().backward()
    assert torch.equal(x.grad, op.embedding_dx(w, ids, 50, 3.0, padding_idx=2))
    x.grad = None
    op.embedding(x, ids).sum().backward()  # a gradient that is broadcast
    assert torch.equal(x.grad, op.embedding_dx(torch.ones(4, 9, 24, device="cuda"), ids, 50))
    # differences: a lookup is linear
    e = torch.zeros_like(x)
    e[7, 5] = 1.0
    d = ((op.embedding(x.detach() + e, ids).double() - op.embedding(x.detach() - e, ids).double()) / 2).sum()
    assert abs(float(d) - float(x.grad[7, 5])) < 1e-4
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(op.embedding(x, ids).pow(2).sum(), x, create_graph=True)[0].sum(), x)


def test_refusals_on_the_gpu():
    x, ids = torch.zeros(5, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    dy = torch.zeros(3, 8, device="cuda")
    for call in (lambda: op.embedding(x[0], ids), lambda: op.embedding(x.t(), ids), lambda: op.embedding(x, ids.cpu()),
                 lambda: op.embedding(x, ids, out=torch.zeros(3, 9, device="cuda")), lambda: op.embedding(x, ids, out=x[:3]),
                 lambda: op.embedding(x, ids, out=torch.zeros(3, 8, device="cuda", dtype=F16)),
                 lambda: op.embedding(x.clone().requires_grad_(), ids, out=dy),
                 lambda: op.embedding_dx(dy, ids[:2], 5), lambda: op.embedding_dx(dy, ids, -1),
                 lambda: op.embedding_dx(dy, ids, 5, accumulate=True), lambda: op.embedding_dx(dy, ids, 3, out=dy),
                 lambda: op.embedding_dx(dy, ids, 5, out=torch.zeros(5, 8, device="cuda").t()),
                 lambda: op.embedding_dx(dy, ids, 5, out=torch.zeros(4, 8, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: op.embedding(x, dy), lambda: op.embedding(x.double(), ids), lambda: op.embedding(x, ids, dtype=torch.int32),
                 lambda: op.embedding_dx(dy, ids.to(torch.int16), 5), lambda: op.embedding_dx(dy, ids, 5, dtype=torch.float64)):
        with pytest.raises(TypeError):
            call()
    lib = _lib.load()  # a workspace that is too small
    assert lib.rafb200_embedding_dx(dy.data_ptr(), 0, ids.data_ptr(), _lib.I64, 3, 5, 8, 1.0, -1, 0, x.data_ptr(), 0, dy.data_ptr(),
                                    16, None) == 1


def test_forward_mode_and_lazy_signs_are_refused():
    """Tensors whose tangent, or whose sign, is not at their address."""
    import torch.autograd.forward_ad as fwd

    x, ids = torch.randn(5, 8, device="cuda"), torch.randint(0, 5, (3,), device="cuda")
    dy, into = torch.randn(3, 8, device="cuda"), torch.zeros(5, 8, device="cuda")

    def calls(x, dy, into):
        return ([lambda: op.embedding(x, ids), lambda: op.embedding(x, ids, out=torch.empty(3, 8, device="cuda")),
                 lambda: op.embedding(x, ids, stream=torch.cuda.current_stream())],
                [lambda: op.embedding_dx(dy, ids, 5), lambda: op.embedding_dx(dy, ids, 5, stream=torch.cuda.current_stream())],
                [lambda: op.embedding_dx(torch.ones(3, 8, device="cuda"), ids, 5, out=into, accumulate=True)])

    with fwd.dual_level():
        for call in sum(calls(*(fwd.make_dual(t, torch.ones_like(t)) for t in (x, dy, into))), []):
            with pytest.raises(ValueError, match="forward"):
                call()
        with torch.no_grad(), pytest.raises(ValueError, match="forward"):
            op.embedding(fwd.make_dual(x, torch.ones_like(x)), ids)
        with pytest.raises(ValueError, match="forward"):
            op.embedding(fwd.make_dual(x.clone().requires_grad_(), torch.ones_like(x)), ids)
        assert torch.equal(op.embedding(x, ids), x[ids])
    assert bool((into == 0).all())
    for call in sum(calls(*map(torch._neg_view, (x, dy, into))), []):
        with pytest.raises(ValueError, match="negat"):
            call()


def test_a_gradient_is_not_cut_off_without_a_word():
    """embedding_dx has no backward, and what is written into out has none either."""
    ids, dy, dx = torch.randint(0, 5, (3,), device="cuda"), torch.randn(3, 8, device="cuda"), torch.zeros(5, 8, device="cuda")
    leaf, out = dy.clone().requires_grad_(), dx.clone().requires_grad_()
    for call in (lambda: op.embedding_dx(leaf, ids, 5), lambda: op.embedding_dx(leaf * 2, ids, 5, out=dx), lambda: op.embedding_dx(dy, ids, 5, out=out),
                 lambda: op.embedding_dx(dy, ids, 5, out=out * 2, accumulate=True), lambda: op.embedding(dx, ids, out=leaf),
                 lambda: op.embedding_dx(leaf, ids, 5, stream=torch.cuda.current_stream())):
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        assert torch.equal(op.embedding_dx(leaf, ids, 5, out=out), op.embedding_dx(dy, ids, 5))


@pytest.mark.parametrize("rows", [255, 256, 511, 512, 513, 262143, 262144, 262145, (1 << 27) - 1])
@pytest.mark.parametrize("n", [4096, 4097, 9999])
def test_every_digit_of_an_id_is_sorted(n, rows):
    """Tables at the borders of the sort's digits, with as many tokens as are ranked by comparison and with more."""
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
    ids[::3] = torch.tensor([rows - 1, 0, rows // 2, rows - 1, rows, -1, 1, rows - 2], device="cuda").repeat(n)[:ids[::3].numel()]
    dy = torch.randn(n, 1 if rows > 1 << 20 else 3, generator=g, device="cuda")
    got = op.embedding_dx(dy, ids, rows)
    check_gradient(got, dy, ids, rows, 1.0)
    assert torch.equal(got, op.embedding_dx(dy, ids, rows))
