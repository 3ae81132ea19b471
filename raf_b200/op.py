"""Python mirror of the RAF operators on the ZeRO optimizer path.

Same names, argument order and dtype rules as ``raf.op.*`` / ``raf._op.imp``
in the reference (``scripts/src_codegen/def_schema.py:525-536,671-738``), on
``torch`` CUDA tensors.  Every function forwards device pointers to the C ABI
(``include/raf_b200.h``); nothing here computes on the host.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import List, Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import BF16, F16, F32, I32, I64, check

_CODES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_NAMES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def dtype_code(dtype) -> int:
    if isinstance(dtype, str):
        dtype = _NAMES[dtype]
    try:
        return _CODES[dtype]
    except KeyError as exc:
        raise TypeError(f"NotImplementedError: {dtype}") from exc


def torch_dtype(dtype):
    return _NAMES[dtype] if isinstance(dtype, str) else dtype


def _check_cuda(*tensors):
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("raf_b200 operators need CUDA tensors; there is no CPU path")
        if not t.is_contiguous():
            raise ValueError("tensors must be compact (contiguous), as in the reference")


def stream_ptr(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    # the address alone: torch.cuda.current_stream() builds a Stream object (3 us a call)
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _raw(stream):
    """The address of a stream, or None: the native module looks up the current one itself."""
    return None if stream is None else stream.cuda_stream


# --------------------------------------------------------------------------- lists
class TensorList:
    """Device-resident tensor list ([g..., p..., m..., v...] of raf.op.lans)."""

    def __init__(self, numels: Sequence[int], g_dtype, out_dtype=torch.float32):
        self.k = len(numels)
        self.numels = [int(n) for n in numels]
        self.g_dtype = torch_dtype(g_dtype)
        self.out_dtype = torch_dtype(out_dtype)
        h = C.c_void_p()
        check(_lib.load().rafb200_tensor_list_create(
            self.k, _lib.i64_array(self.numels), dtype_code(self.g_dtype),
            dtype_code(self.out_dtype), C.byref(h)))
        self.handle = h
        self._keep = None
        self._ws = None

    def bind(self, g, p, m, v=None, out=None, stream=None):
        def ptrs(ts, dtype):
            if ts is None:
                return None
            assert len(ts) == self.k
            res = []
            for t, n in zip(ts, self.numels):
                if t is None:
                    res.append(0)
                    continue
                _check_cuda(t)
                assert t.numel() == n and t.dtype == dtype, (t.shape, t.dtype, n, dtype)
                res.append(t.data_ptr())
            return _lib.ptr_array(res)

        check(_lib.load().rafb200_tensor_list_bind(
            self.handle, ptrs(g, self.g_dtype), ptrs(p, torch.float32), ptrs(m, torch.float32),
            ptrs(v, torch.float32), ptrs(out, self.out_dtype), stream_ptr(stream)))
        self._keep = (g, p, m, v, out)  # the device table holds raw pointers

    def tune(self, lead_elems=8 << 20, gap_items=0, max_blocks=0):
        """Scheduling knobs of the LANS kernel (rafb200_tensor_list_tune); the defaults are
        the ones a list is created with."""
        check(_lib.load().rafb200_tensor_list_tune(self.handle, int(lead_elems), int(gap_items),
                                                   int(max_blocks)))

    def set_wait_limit(self, limit_ms: int):
        """Bound of every wait inside the LANS kernel (default 2 s)."""
        check(_lib.load().rafb200_tensor_list_set_wait_limit(self.handle, int(limit_ms)))

    def set_symmetric(self, rank, g_peers, p_peers, g_offsets_bytes, g_mc=0, p_mc=0, reduce_scatter=True,
                      all_gather=True):
        """The collectives inside the update kernels (rafb200_tensor_list_set_symmetric):
        ``g_peers`` / ``p_peers`` = every rank's gradient / parameter buffer as addressable here
        (device addresses), ``g_offsets_bytes`` = each tensor's offset inside the gradient buffer."""
        world = len(g_peers)
        off = _lib.i64_array([int(x) for x in g_offsets_bytes])
        check(_lib.load().rafb200_tensor_list_set_symmetric(
            self.handle, world, int(rank), _lib.ptr_array([int(x) for x in g_peers]), int(g_mc) or None,
            _lib.ptr_array([int(x) for x in p_peers]), int(p_mc) or None, off, int(bool(reduce_scatter)),
            int(bool(all_gather))))

    def set_lans_items(self, items):
        """Replace the LANS work-item table: ``items`` is an (n, 2) uint32 array."""
        import numpy as np

        a = np.ascontiguousarray(items, np.uint32).reshape(-1, 2)
        check(_lib.load().rafb200_tensor_list_set_lans_items(self.handle, a.ctypes.data, a.shape[0]))

    def lans_workspace(self) -> torch.Tensor:
        if self._ws is None:
            n = _lib.load().rafb200_lans_workspace_bytes(self.handle)
            self._ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        return self._ws

    def close(self):
        if self.handle:
            torch.cuda.synchronize()
            _lib.load().rafb200_tensor_list_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter shutdown
            pass


# --------------------------------------------------------------------------- optimizers
def sgd(x, dx, v, learning_rate, mu):
    """raf.op.sgd: returns (v1, x1) as NEW tensors (src/op/declare/optimizer.cc:22-44)."""
    r = _lib.ops().sgd(x, dx, v, learning_rate, mu)
    if r.__class__ is tuple:
        return r
    if r is not None:
        check(r)
    _check_cuda(x, dx, v)
    if x.shape != dx.shape or x.shape != v.shape:
        raise ValueError("sgd: x, dx and v must have the same shape")
    x1 = x.clone()
    v1 = v.clone()
    sgd_(x1, dx, v1, learning_rate, mu)
    return v1, x1


def sgd_(x, dx, v, learning_rate, mu, weight_decay=0.0, grad_scale=1.0, out=None, stream=None):
    """In-place fused form: x, v fp32; dx fp32/fp16/bf16; out (optional) receives cast(x1)."""
    _check_cuda(x, dx, v)
    assert x.dtype == torch.float32 and v.dtype == torch.float32
    if out is not None:
        _check_cuda(out)
        assert out.numel() == x.numel()
    check(_lib.load().rafb200_sgd(
        x.data_ptr(), dx.data_ptr(), dtype_code(dx.dtype), v.data_ptr(), x.numel(),
        float(learning_rate), float(mu), float(weight_decay), float(grad_scale),
        out.data_ptr() if out is not None else None,
        dtype_code(out.dtype) if out is not None else F32, stream_ptr(stream)))
    return x, v


def sgd_list_(tl: TensorList, learning_rate, mu, weight_decay=0.0, grad_scale=1.0, stream=None):
    check(_lib.load().rafb200_sgd_list(tl.handle, float(learning_rate), float(mu),
                                       float(weight_decay), float(grad_scale), stream_ptr(stream)))


def lans_list_(tl: TensorList, step, learning_rate, beta1, beta2, eps, bias_correction,
               weight_decay, grad_averaging, mode, normalize_grad, grad_scale=1.0, stream=None):
    """raf.op.lans on a bound TensorList; ``step`` is an int or a 0-d fp32 CUDA tensor."""
    ws = tl.lans_workspace()
    step_dev = None
    if isinstance(step, torch.Tensor):
        assert step.is_cuda and step.dtype == torch.float32 and step.dim() == 0
        step_dev, step = step.data_ptr(), 0
    check(_lib.load().rafb200_lans(
        tl.handle, int(step), step_dev, float(learning_rate), float(beta1), float(beta2),
        float(eps), int(bias_correction), float(weight_decay), int(grad_averaging), int(mode),
        int(bool(normalize_grad)), float(grad_scale), ws.data_ptr(), ws.numel(),
        stream_ptr(stream)))


def lans_status(tl: TensorList, want_norms=False, stream=None):
    """Waits for the stream; raises if a bounded device wait expired; returns norms[k,4] or None."""
    import numpy as np

    norms = np.zeros((tl.k, 4), np.float32) if want_norms else None
    check(_lib.load().rafb200_lans_status(
        tl.handle, tl.lans_workspace().data_ptr(),
        norms.ctypes.data if norms is not None else None, stream_ptr(stream)))
    return norms


def lans(tensor_list: List[torch.Tensor], step, learning_rate, beta1, beta2, eps, bias_correction,
         weight_decay, grad_averaging, mode, normalize_grad):
    """raf.op.lans (python/raf/optim/lans.py:87-99): tensor_list = g + p + m + v, updated in place.

    Like the reference (src/op/dialect/cuda/lans.cc:38-40) it takes fp32 tensors only;
    16-bit gradients go through :class:`TensorList` / :func:`lans_list_`.
    """
    done = _lib.ops().lans(tensor_list, step, learning_rate, beta1, beta2, eps, bias_correction, weight_decay,
                           grad_averaging, mode, normalize_grad)
    if done is True:
        return tensor_list
    if done is not None:
        check(done)
    n = len(tensor_list)
    if n % 4 != 0:
        raise ValueError("lans: tensor_list must hold g, p, m and v lists of equal length")
    k = n // 4
    for t in tensor_list:
        _check_cuda(t)
        if t.dtype != torch.float32:
            raise TypeError("LANS only takes FP32 inputs")
    g, p, m, v = (tensor_list[i * k:(i + 1) * k] for i in range(4))
    tl = TensorList([t.numel() for t in p], torch.float32, torch.float32)
    try:
        tl.bind(g, p, m, v)
        lans_list_(tl, step, learning_rate, beta1, beta2, eps, bias_correction, weight_decay,
                   grad_averaging, mode, normalize_grad)
        lans_status(tl)
    finally:
        tl.close()
    return tensor_list


def adam_list_(tl: TensorList, step, learning_rate, beta1, beta2, eps, bias_correction,
               weight_decay, mode, grad_scale=1.0, stream=None):
    """Adam / AdamW on a bound TensorList (no reference operator; see include/raf_b200.h)."""
    check(_lib.load().rafb200_adam(
        tl.handle, int(step), None, float(learning_rate), float(beta1), float(beta2), float(eps),
        int(bias_correction), float(weight_decay), int(mode), float(grad_scale),
        stream_ptr(stream)))


# --------------------------------------------------------------------------- casts, packing
def cast(data, dtype, out=None, stream=None):
    """raf.op.cast."""
    _check_cuda(data)
    dtype = torch_dtype(dtype)
    if out is None:
        out = torch.empty_like(data, dtype=dtype)
    check(_lib.load().rafb200_cast(data.data_ptr(), dtype_code(data.dtype), out.data_ptr(),
                                   dtype_code(dtype), data.numel(), stream_ptr(stream)))
    return out


def group_cast(tensor_list, dtype, stream=None):
    """raf.op.group_cast: one launch for the whole tuple."""
    dtype = torch_dtype(dtype)
    r = _lib.ops().group_cast(tensor_list, _CODES.get(dtype, -1), _raw(stream))
    if r.__class__ is list:
        return r
    if r is not None:
        check(r)
    if not tensor_list:
        return []
    _check_cuda(*tensor_list)
    src_dtype = tensor_list[0].dtype
    assert all(t.dtype == src_dtype for t in tensor_list)
    outs = [torch.empty_like(t, dtype=dtype) for t in tensor_list]
    check(_lib.load().rafb200_group_cast(
        len(tensor_list), _lib.ptr_array([t.data_ptr() for t in tensor_list]),
        dtype_code(src_dtype), _lib.ptr_array([t.data_ptr() for t in outs]), dtype_code(dtype),
        _lib.i64_array([t.numel() for t in tensor_list]), stream_ptr(stream)))
    return outs


def fuse_tensor(tensor_list, stream=None):
    """raf.op.fuse_tensor: concatenate a tuple into one flat buffer."""
    r = _lib.ops().fuse_tensor(tensor_list, _raw(stream))
    if isinstance(r, torch.Tensor):
        return r
    if r is not None:
        check(r)
    _check_cuda(*tensor_list)
    dtype = tensor_list[0].dtype
    numels = [t.numel() for t in tensor_list]
    offsets = [0]
    for n in numels[:-1]:
        offsets.append(offsets[-1] + n)
    flat = torch.empty(sum(numels), dtype=dtype, device=tensor_list[0].device)
    check(_lib.load().rafb200_fuse_tensor(
        len(tensor_list), _lib.ptr_array([t.data_ptr() for t in tensor_list]),
        _lib.i64_array(numels), _lib.i64_array(offsets), flat.element_size(), flat.data_ptr(),
        stream_ptr(stream)))
    return flat


def defuse_tensor(data, sizes, shapes, shape_indices, stream=None):
    """raf.op.defuse_tensor (schema DefuseTensorArgs{data, sizes, shapes, shape_indices})."""
    r = _lib.ops().defuse_tensor(data, sizes, shapes, shape_indices, _raw(stream))
    if r.__class__ is list:
        return r
    if r is not None:
        check(r)
    _check_cuda(data)
    outs, offsets, start = [], [], 0
    off = 0
    for i, n in enumerate(sizes):
        shape = tuple(shapes[start:shape_indices[i]])
        start = shape_indices[i]
        outs.append(torch.empty(shape, dtype=data.dtype, device=data.device))
        assert outs[-1].numel() == n
        offsets.append(off)
        off += n
    if off > data.numel():
        raise ValueError(f"defuse_tensor: sizes hold {off} elements, data {data.numel()}")
    check(_lib.load().rafb200_defuse_tensor(
        len(outs), _lib.ptr_array([t.data_ptr() for t in outs]), _lib.i64_array(sizes),
        _lib.i64_array(offsets), data.element_size(), data.data_ptr(), stream_ptr(stream)))
    return outs


# --------------------------------------------------------------------------- the two ends of a model
_INDEX = {torch.int64: I64, torch.int32: I32}


def _index_code(t) -> int:
    try:
        return _INDEX[t.dtype]
    except KeyError as exc:
        raise TypeError(f"indices are int32 or int64, not {t.dtype}") from exc


def _same_device(*tensors):
    if any(t.device != tensors[0].device for t in tensors):
        raise ValueError("tensors must be on one device")


def _check_values(what, *tensors):
    """Tensors whose sign or tangent is not at their address: what is computed from there would be without it."""
    for t in tensors:
        if t is None:
            continue
        if t.is_neg():
            raise ValueError(f"{what}: a tensor that is still to be negated; resolve_neg() it first")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what}: there are no forward-mode derivatives, and a tensor has a tangent")


def _check_no_graph(what, name, t):
    if torch.is_grad_enabled() and t is not None and t.requires_grad:
        raise ValueError(f"{what}: the result is part of no autograd graph, and {name} requires a gradient; detach it")


def _span(t):
    """The bytes a tensor of positive strides reaches over."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _check_apart(out, *inputs):
    lo, hi = _span(out)
    for t in inputs:
        a, b = _span(t)
        if a < hi and lo < b:
            raise ValueError("out overlaps an input")


@contextlib.contextmanager
def _launching(t, stream, *others):
    """On the tensor's device and the given stream, for allocations too: what a call allocates there is not
    handed to another stream's work while the call still runs, nor are the tensors it is given."""
    if stream is not None and stream.device != t.device:
        raise ValueError("the stream belongs to another device than the tensors")
    with torch.cuda.device(t.device), torch.cuda.stream(stream):
        if stream is not None and not torch.cuda.is_current_stream_capturing():
            for x in (t,) + others:
                if x is not None:
                    x.record_stream(stream)
        yield torch._C._cuda_getCurrentRawStream(t.device.index)


def _check_capturable(name, x):
    """Before a node is put behind x: what backward could not be captured through is refused here, where an exception is one."""
    if not torch.cuda.is_current_stream_capturing():
        return
    reaches = _lib.ops().reaches_default_stream(x)
    if reaches is None:  # the stream of a node is not to be had from Python
        raise RuntimeError(f"{name}: under capture, whether a backward could be captured is known to the native module alone, and "
                           "raf_b200._ops is not available; detach the input, or build the module")
    if reaches:
        raise RuntimeError(f"{name}: under capture, but the input's autograd graph reaches into one that was built on the default "
                           "stream and still lives, so its backward cannot be captured; drop that graph first, or detach the input")


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, indices, scale, padding_idx, dtype):
        ctx.save_for_backward(indices)
        ctx.how = x.shape[0], scale, padding_idx, x.dtype
        return embedding(x.detach(), indices, scale, padding_idx, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        num_weight, scale, padding_idx, dtype = ctx.how
        return embedding_dx(dy.contiguous(), *ctx.saved_tensors, num_weight, scale, padding_idx, dtype), None, None, None, None


def embedding(x, indices, scale=1.0, padding_idx=None, dtype=None, out=None, stream=None):
    """raf.op.embedding(x, indices), times ``scale``: ``out[..., :] = scale * x[indices[...], :]``.

    ``x`` is [rows, width] in fp32 / fp16 / bf16, ``indices`` any shape of int32 / int64; the result is of ``dtype``
    (default: x's), rounded once.  An index outside [0, rows) reads as a row of zeros.  Where ``x`` requires a
    gradient, backward is :func:`embedding_dx`, for which ``padding_idx`` names an index that counts nothing.  Forward and
    backward may be captured in one graph while no eager graph of the same leaves lives; else, and where raf_b200._ops, which
    looks for one, is missing, the captured call is refused.
    """
    if out is None and stream is None:
        r = _lib.ops().embedding(x, indices, scale, dtype)
        if isinstance(r, torch.Tensor):
            return r
        if r is not None:
            check(r)
    _check_cuda(x, indices)
    _same_device(x, indices)
    _check_values("embedding", x, out)
    _check_no_graph("embedding", "out", out)
    if x.dim() != 2:
        raise ValueError("embedding: x is a table, [rows, width]")
    dtype = x.dtype if dtype is None else torch_dtype(dtype)
    code, out_code, index = dtype_code(x.dtype), dtype_code(dtype), _index_code(indices)
    if torch.is_grad_enabled() and x.requires_grad:
        if out is not None:
            raise ValueError("embedding: out has no gradient; x must not require one")
        with _launching(x, stream, indices):  # autograd runs backward on the stream that is current here
            _check_capturable("embedding", x)
            return _Embedding.apply(x, indices, scale, padding_idx, dtype)
    shape = indices.shape + x.shape[1:]
    if out is not None:
        _check_cuda(out)
        _same_device(x, out)
        if out.shape != shape or out.dtype != dtype:
            raise ValueError(f"embedding: out is to be {tuple(shape)} of {dtype}")
        _check_apart(out, x, indices)
        torch.autograd.graph.increment_version(out)
    with _launching(x, stream, indices, out) as raw:
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=x.device)
        check(_lib.load().rafb200_embedding(x.data_ptr(), code, x.shape[0], x.shape[1], indices.data_ptr(), index,
                                            indices.numel(), float(scale), out.data_ptr(), out_code, raw))
    return out


def embedding_dx(dy, indices, num_weight, scale=1.0, padding_idx=None, dtype=None, out=None, accumulate=False, stream=None):
    """raf.op.embedding_dx(dy, indices, num_weight): the gradient [num_weight, width] of the table,
    ``dx[r, :] = scale * sum of dy[i, :] over indices[i] == r``, in ``dtype`` (default: dy's, or out's).

    ``out`` takes the result: a gradient that an optimizer or ZeroStep reads.  With ``accumulate`` the sums are
    added to it (a further micro-batch, a matrix product that shares the table), rounded once to its type, and rows
    without a token stay as they are.  Indices equal to ``padding_idx`` or outside [0, num_weight) count nothing (a negative
    ``padding_idx`` names no row).
    The same call gives the same bits: sums run in an order that the indices fix.  The result is data, part of no autograd graph:
    ``dy`` and ``out`` must not require a gradient.
    """
    if stream is None:
        r = _lib.ops().embedding_dx(dy, indices, num_weight, scale, padding_idx, dtype, out, accumulate)
        if isinstance(r, torch.Tensor):
            return r
        if r is not None:
            check(r)
    _check_cuda(dy, indices)
    _same_device(dy, indices)
    _check_values("embedding_dx", dy, out)
    _check_no_graph("embedding_dx", "dy", dy)
    _check_no_graph("embedding_dx", "out", out)
    if dy.dim() != indices.dim() + 1 or dy.shape[:-1] != indices.shape:
        raise ValueError("embedding_dx: dy has the shape of indices and one dimension more")
    num_weight, width = int(num_weight), dy.shape[-1]
    if num_weight < 0:
        raise ValueError("embedding_dx: negative num_weight")
    if dtype is None:
        dtype = dy.dtype if out is None else out.dtype
    dtype = torch_dtype(dtype)
    code, out_code, index = dtype_code(dy.dtype), dtype_code(dtype), _index_code(indices)
    if out is None:
        if accumulate:
            raise ValueError("embedding_dx: accumulate needs the gradient to add to, out")
    else:
        _check_cuda(out)
        _same_device(dy, out)
        if out.shape != (num_weight, width) or out.dtype != dtype:
            raise ValueError(f"embedding_dx: out is to be {(num_weight, width)} of {dtype}")
        _check_apart(out, dy, indices)
        torch.autograd.graph.increment_version(out)
    # outside [0, num_weight): nothing is left out
    padding_idx = -1 if padding_idx is None else int(padding_idx)
    lib, n = _lib.load(), indices.numel()
    with _launching(dy, stream, indices, out) as raw:
        if out is None:
            out = torch.empty((num_weight, width), dtype=dtype, device=dy.device)
        ws = torch.empty(lib.rafb200_embedding_dx_workspace_bytes(n, width), dtype=torch.uint8, device=dy.device)
        check(lib.rafb200_embedding_dx(dy.data_ptr(), code, indices.data_ptr(), index, n, num_weight, width, float(scale),
                                       padding_idx, int(bool(accumulate)), out.data_ptr(), out_code, ws.data_ptr(),
                                       ws.numel(), raw))
    return out


def _rows_of(t, what):
    """[..., v] as [n, v] with consecutive elements in a row, not copied."""
    if not t.is_cuda:
        raise ValueError("raf_b200 operators need CUDA tensors; there is no CPU path")
    if t.dim() < 1:
        raise ValueError(f"{what}: at least one dimension")
    v = t.shape[-1]
    try:
        rows = t.view(-1 if t.numel() else t.shape[:-1].numel(), v)
    except RuntimeError as exc:
        raise ValueError(f"{what}: rows must lie at one distance from each other") from exc
    if (v > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < v):
        raise ValueError(f"{what}: a row's elements must be consecutive, and rows must not overlap")
    return rows, (rows.stride(0) if rows.shape[0] > 1 else v)


def _distill_args(pred, teacher_logits, teacher_ids, labels, temperature, alpha, ignore_index):
    rows, ld = _rows_of(pred, "pred")
    given = [teacher_logits, teacher_ids] + ([] if labels is None else [labels])
    _check_cuda(*given)
    _same_device(pred, *given)
    _check_values("distill_loss", pred, teacher_logits)
    lead = pred.shape[:-1]
    if teacher_logits.dim() != pred.dim() or teacher_logits.shape[:-1] != lead or teacher_ids.shape != teacher_logits.shape:
        raise ValueError("distill_loss: teacher_logits and teacher_ids have pred's shape up to the last dimension, and each other's")
    if labels is not None and labels.shape != lead:
        raise ValueError("distill_loss: labels have pred's shape without the last dimension")
    if rows.shape[1] == 0 and rows.shape[0]:
        raise ValueError("distill_loss: no classes")
    if labels is None and alpha != 1.0:
        raise ValueError("distill_loss: alpha below 1 needs labels")
    return _lib.Distill(
        pred.data_ptr(), teacher_logits.data_ptr(), teacher_ids.data_ptr(), labels.data_ptr() if labels is not None else None,
        rows.shape[0], max(rows.shape[1], 1), max(ld, 1), int(ignore_index), float(temperature), float(alpha),
        teacher_logits.shape[-1], dtype_code(pred.dtype), dtype_code(teacher_logits.dtype), _index_code(teacher_ids),
        _index_code(labels) if labels is not None else I64)


def _weights_of(dy, pred):
    """The address and step of the rows' weights."""
    if dy is None:
        return None, 0
    _check_cuda(dy)
    _same_device(pred, dy)
    _check_values("distill_loss", dy)
    if dy.dtype != torch.float32:
        raise TypeError("dy is fp32")
    if dy.dim() == 0:
        return dy.data_ptr(), 0
    if dy.shape != pred.shape[:-1]:
        raise ValueError("dy has pred's shape without the last dimension, or none")
    return dy.data_ptr(), 1


def _gradient_for(pred, out, others):
    if out is None:
        return torch.empty(pred.shape, dtype=pred.dtype, device=pred.device), pred.shape[-1]
    rows, ld = _rows_of(out, "out")
    _same_device(pred, out)
    _check_values("distill_loss", out)
    if out is not pred:
        _check_no_graph("distill_loss", "out", out)
    if out.shape != pred.shape or out.dtype != pred.dtype:
        raise ValueError(f"out is to be {tuple(pred.shape)} of {pred.dtype}")
    _check_apart(out, *(t for t in others if t is not None))
    torch.autograd.graph.increment_version(out)
    return out, ld


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, teacher_logits, teacher_ids, labels, temperature, alpha, ignore_index):
        loss, stats = distill_loss(pred.detach(), teacher_logits, teacher_ids, labels, temperature, alpha, ignore_index)
        ctx.save_for_backward(pred, teacher_logits, teacher_ids, stats, labels)
        ctx.how = temperature, alpha, ignore_index
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        return (distill_loss_dpred(dy.contiguous(), *ctx.saved_tensors, *ctx.how),) + (None,) * 6


def distill_loss(pred, teacher_logits, teacher_ids, labels=None, temperature=1.0, alpha=1.0, ignore_index=-100, stream=None):
    """Loss of ``pred`` [..., v] against a teacher's top logits, per row: (loss [...], stats [..., 4]), fp32.

    ``alpha T^2 sum p (log p - log softmax(pred / T)) + (1 - alpha) (-log softmax(pred)[label])`` with p the softmax of
    the row's ``teacher_logits / T`` [..., k <= 1024] over the classes ``teacher_ids``; an entry whose class is outside
    [0, v) is absent.  Without ``labels`` alpha is 1.  A row whose label is ``ignore_index`` or outside [0, v) has loss
    and gradient 0.  Rows of ``pred`` may lie further apart than v (logits padded for a matrix product).

    ``stats`` is what :func:`distill_loss_dpred` takes: a row's maximum, sum of ``exp((pred - max) / T)``, sum of
    ``exp(pred - max)``, and a value that it does not read.  What this loss does not sum up is NaN, and so is a gradient that
    takes it: the last sum where T is not 1 and there is no hard term, all of them in a row that its label leaves out.  Where
    ``pred`` requires a gradient, backward calls it; for a captured backward the condition of :func:`embedding` holds.
    """
    if stream is None:
        r = _lib.ops().distill(None, pred, teacher_logits, teacher_ids, None, labels, temperature, alpha, ignore_index, 1.0, 0)
        if r.__class__ is tuple:
            return r
        if r is not None:
            check(r)
    d = _distill_args(pred, teacher_logits, teacher_ids, labels, temperature, alpha, ignore_index)
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise ValueError("distill_loss: the teacher gets no gradient; detach its logits")
    if torch.is_grad_enabled() and pred.requires_grad:
        with _launching(pred, stream, teacher_logits, teacher_ids, labels):
            _check_capturable("distill_loss", pred)
            return _DistillLoss.apply(pred, teacher_logits, teacher_ids, labels, temperature, alpha, ignore_index)
    with _launching(pred, stream, teacher_logits, teacher_ids, labels) as raw:
        loss = torch.empty(pred.shape[:-1], dtype=torch.float32, device=pred.device)
        stats = torch.empty(pred.shape[:-1] + (4,), dtype=torch.float32, device=pred.device)
        check(_lib.load().rafb200_distill_loss(C.byref(d), loss.data_ptr(), stats.data_ptr(), raw))
    return loss, stats


def distill_loss_dpred(dy, pred, teacher_logits, teacher_ids, stats, labels=None, temperature=1.0, alpha=1.0, ignore_index=-100,
                       grad_scale=1.0, out=None, stream=None):
    """Gradient of :func:`distill_loss`: ``dy * grad_scale * d loss / d pred``, of pred's shape and type.

    ``dy`` is fp32, one weight per row, one for all rows (0-dimensional), or None for 1; ``grad_scale`` is the loss scale that
    the optimizers' own ``grad_scale`` takes back.  ``out`` takes the result and may be ``pred`` itself; another one must not
    require a gradient.  The result is data, part of no autograd graph.
    """
    if out is None and stream is None:
        r = _lib.ops().distill(dy, pred, teacher_logits, teacher_ids, stats, labels, temperature, alpha, ignore_index, grad_scale, 1)
        if isinstance(r, torch.Tensor):
            return r
        if r is not None:
            check(r)
    d = _distill_args(pred, teacher_logits, teacher_ids, labels, temperature, alpha, ignore_index)
    weights, step = _weights_of(dy, pred)
    _check_cuda(stats)
    _same_device(pred, stats)
    _check_values("distill_loss", stats)
    if stats.shape != pred.shape[:-1] + (4,) or stats.dtype != torch.float32:
        raise ValueError("distill_loss_dpred: stats are those of distill_loss for this pred")
    with _launching(pred, stream, dy, teacher_logits, teacher_ids, stats, labels, out) as raw:
        out, ld = _gradient_for(pred, out, (dy, teacher_logits, teacher_ids, stats, labels))
        check(_lib.load().rafb200_distill_loss_dpred(C.byref(d), weights, step, float(grad_scale), stats.data_ptr(),
                                                     out.data_ptr(), ld, raw))
    return out


def distill_loss_with_dpred(dy, pred, teacher_logits, teacher_ids, labels=None, temperature=1.0, alpha=1.0, ignore_index=-100,
                            grad_scale=1.0, out=None, stream=None):
    """:func:`distill_loss` and :func:`distill_loss_dpred` in one pass over the logits, where the rows' weights ``dy`` are
    known beforehand: (loss, dpred).  Both are data, part of no autograd graph."""
    if out is None and stream is None:
        r = _lib.ops().distill(dy, pred, teacher_logits, teacher_ids, None, labels, temperature, alpha, ignore_index, grad_scale, 2)
        if r.__class__ is tuple:
            return r
        if r is not None:
            check(r)
    d = _distill_args(pred, teacher_logits, teacher_ids, labels, temperature, alpha, ignore_index)
    weights, step = _weights_of(dy, pred)
    with _launching(pred, stream, dy, teacher_logits, teacher_ids, labels, out) as raw:
        loss = torch.empty(pred.shape[:-1], dtype=torch.float32, device=pred.device)
        out, ld = _gradient_for(pred, out, (dy, teacher_logits, teacher_ids, labels))
        check(_lib.load().rafb200_distill_loss_with_dpred(C.byref(d), weights, step, float(grad_scale), loss.data_ptr(),
                                                          out.data_ptr(), ld, raw))
    return loss, out
