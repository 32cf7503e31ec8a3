"""Operators of latent factors on device tensors: row lookup with its gradient (blp_lookup*), the
softmax loss over the whole catalogue with its gradients (blp_softmax_loss*), and scores of the catalogue
from 8-bit factors (blp_quantize_rows, blp_scores8) -- all in blp.h.

They stand beside :class:`blp.factor.DeviceSVD`, whose factors they read, train and score: rows of a
user table and of a business table, ``k`` components a row. Every argument that holds data is a torch
tensor on one GPU, its rows contiguous (a row stride larger than the row is fine); the work is queued
on torch's current stream of that device, workspaces come from torch's allocator, and nothing waits
for the device. Wrong arguments raise ValueError before anything is queued.
"""
import ctypes

from . import _lib
from ._lib import check, lib

_P, _I64, _I32, _F = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
_PI64 = ctypes.POINTER(ctypes.c_int64)
_lib.register("blp_softmax_loss_workspace", [_I32, _P, _I64, _P, _I64, _I64, _I64, _I32, _I32, _I32, _PI64])
_lib.register("blp_softmax_loss", [_I32, _P, _I32, _P, _I64, _P, _I64, _P, _I32, _I64, _I64, _I32, _F, _P, _P, _P, _I32,
                                   _I32, _P, _I64, _P, _I64, _P, _I64])
_lib.register("blp_softmax_loss_backward", [_I32, _P, _I32, _P, _I64, _P, _I64, _P, _I32, _I64, _I64, _I32, _F, _P, _P,
                                            _I32, _P, _P, _I64, _P, _I64, _P, _I64])
_lib.register("blp_lookup", [_I32, _P, _I32, _P, _I64, _I64, _I32, _P, _I32, _I64, _F, _P, _I64])
_lib.register("blp_lookup_grad_workspace", [_I32, _I64, _I64, _I32, _PI64])
_lib.register("blp_lookup_grad", [_I32, _P, _I32, _P, _I64, _P, _I32, _I64, _I64, _I32, _F, _P, _I64, _I32, _P, _I64])
_lib.register("blp_quantize_rows", [_I32, _P, _I32, _P, _I64, _I64, _I32, _P, _I64, _P])
_lib.register("blp_scores8_workspace", [_P, _I64, _P, _I64, _I64, _I64, _I32, _PI64])
_lib.register("blp_scores8", [_I32, _P, _P, _I64, _P, _P, _I64, _P, _I64, _I64, _I32, _I32, _P, _I64, _P, _I64])

_torch = None
_TYPES = {}


def _t():
    """torch, imported on the first call: the graph engine works without it."""
    global _torch
    if _torch is None:
        import torch

        _TYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        _torch = torch
    return _torch


def _rows(t, what, dtypes):
    """`t` as (n, k) rows: a 2-d tensor on a GPU with contiguous rows that do not overlap."""
    torch = _t()
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.dtype not in dtypes or not t.is_cuda:
        raise ValueError("%s must be a 2-d GPU tensor of %s (got %s)" % (
            what, " / ".join(str(d)[6:] for d in dtypes),
            "%s %s on %s" % (tuple(t.shape), t.dtype, t.device) if isinstance(t, torch.Tensor) else type(t)))
    if t.shape[1] < 1 or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError("%s must have contiguous, non-overlapping rows of at least one element (shape %s, strides %s)" % (
            what, tuple(t.shape), tuple(t.stride())))
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ids(t, what, device, n=None):
    torch = _t()
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64) or t.device != device \
            or not t.is_contiguous() or (n is not None and tuple(t.shape) != (n,)):
        raise ValueError("%s must be a contiguous int32 / int64 tensor%s on %s (got %s)" % (
            what, "" if n is None else " of shape (%d,)" % n, device,
            "%s %s on %s" % (tuple(t.shape), t.dtype, t.device) if isinstance(t, torch.Tensor) else type(t)))
    return 1 if t.dtype == torch.int64 else 0


def _stream(device):
    return _torch.cuda.current_stream(device).cuda_stream


_REDUCTIONS = ("mean", "sum", "none")


def _loss_args(x, table, target, scale, reduction):
    torch = _t()
    ldx = _rows(x, "x", tuple(_TYPES))
    ldt = _rows(table, "table", (x.dtype,))
    if table.shape[1] != x.shape[1] or table.device != x.device:
        raise ValueError("x %s and table %s must have rows of the same length on one device" % (
            tuple(x.shape), tuple(table.shape)))
    if table.shape[0] < 1:
        raise ValueError("the catalogue must have at least one row")
    wide = _ids(target, "target", x.device, x.shape[0])
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be one of %s (got %r)" % (", ".join(_REDUCTIONS), reduction))
    return torch, ldx, ldt, wide, _scale(scale)


def _loss_workspace(torch, x, ldx, table, ldt, forward, grads):
    n = ctypes.c_int64(0)
    check(lib().blp_softmax_loss_workspace(_TYPES[x.dtype], x.data_ptr(), ldx, table.data_ptr(), ldt, x.shape[0],
                                           table.shape[0], x.shape[1], forward, grads, ctypes.byref(n)))
    return torch.empty(n.value, dtype=torch.uint8, device=x.device)


def _loss_forward(x, table, target, scale, reduction, grads):
    """-> (loss or total, lse, total, dx, dtable)"""
    torch, ldx, ldt, wide, scale = _loss_args(x, table, target, scale, reduction)
    m, k = x.shape
    stats = torch.empty((2 * m + 2,), dtype=torch.float32, device=x.device)
    loss, lse, total = stats[:m], stats[m:2 * m], stats[2 * m:]
    summed = reduction != "none"
    dx = torch.empty((m, k), dtype=x.dtype, device=x.device) if grads else None
    dt = torch.empty((table.shape[0], k), dtype=x.dtype, device=x.device) if grads else None
    ws = _loss_workspace(torch, x, ldx, table, ldt, 1, 1 if grads else 0)
    check(lib().blp_softmax_loss(
        x.device.index, _stream(x.device), _TYPES[x.dtype], x.data_ptr(), ldx, table.data_ptr(), ldt, target.data_ptr(), wide,
        m, table.shape[0], k, scale, loss.data_ptr(), lse.data_ptr(), total.data_ptr() if summed else None,
        1 if reduction == "mean" else 0, 1 if grads else 0, dx.data_ptr() if grads else None, k,
        dt.data_ptr() if grads else None, k, ws.data_ptr(), ws.numel()))
    return (total[0] if summed else loss), lse, total, dx, dt


def softmax_loss(x, table, target, scale=1.0, reduction="mean"):
    """Softmax cross entropy of ``scale * x @ table.T`` against ``target``, without keeping the scores.

    x (m, k), table (n, k): float32, bfloat16 or float16, the same type; target (m,) int32 / int64: the
    row of `table` that belongs to each row of x. A target outside [0, n) (-1, as in the top-k lists'
    missing slots) ignores its row: loss 0, gradient 0, whatever x holds there. reduction "mean" (over
    the rows not ignored; 0 if there is none), "sum" or "none" (one loss a row). Returns float32;
    differentiable in x and table. Sums and the softmax's statistics are held in 32 bits."""
    torch = _t()
    if torch.is_grad_enabled() and (getattr(x, "requires_grad", False) or getattr(table, "requires_grad", False)):
        return _function("loss").apply(x, table, target, scale, reduction)
    return _loss_forward(x, table, target, scale, reduction, False)[0]


def softmax_loss_grad(x, table, target, scale=1.0, reduction="mean"):
    """-> (loss, dx, dtable): :func:`softmax_loss` ("mean" or "sum") and its gradients in one call, for
    training loops that do not go through autograd."""
    if reduction == "none":
        raise ValueError("softmax_loss_grad: reduction must be mean or sum")
    loss, _, _, dx, dt = _loss_forward(x, table, target, scale, reduction, True)
    return loss, dx, dt


def softmax_loss_backward(grad, lse, count, x, table, target, scale=1.0, need_x=True, need_table=True):
    """-> (dx, dtable) of :func:`softmax_loss`: `grad` float32, one value or one a row; `lse` (m,) the
    forward pass's; `count` a float32 tensor that divides the gradient (mean) or None."""
    torch, ldx, ldt, wide, scale = _loss_args(x, table, target, scale, "none")
    m, k = x.shape
    for t, what, shapes in ((grad, "grad", ((), (1,), (m,))), (lse, "lse", ((m,),)), (count, "count", ((), (1,)))):
        if t is None and what == "count":
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous() \
                or tuple(t.shape) not in shapes:
            raise ValueError("%s must be a contiguous float32 tensor of shape %s on %s" % (what, shapes[-1], x.device))
    stride = 1 if grad.dim() == 1 and m > 1 else 0
    dx = torch.empty((m, k), dtype=x.dtype, device=x.device) if need_x else None
    dt = torch.empty((table.shape[0], k), dtype=x.dtype, device=x.device) if need_table else None
    ws = _loss_workspace(torch, x, ldx, table, ldt, 0, 1)
    check(lib().blp_softmax_loss_backward(
        x.device.index, _stream(x.device), _TYPES[x.dtype], x.data_ptr(), ldx, table.data_ptr(), ldt, target.data_ptr(), wide,
        m, table.shape[0], k, scale, lse.data_ptr(), grad.data_ptr(), stride, None if count is None else count.data_ptr(),
        None if dx is None else dx.data_ptr(), k, None if dt is None else dt.data_ptr(), k, ws.data_ptr(), ws.numel()))
    return dx, dt


def _scale(scale):
    scale = float(scale)
    if not abs(scale) < float("inf"):
        raise ValueError("scale must be finite (got %r)" % scale)
    return scale


def lookup(table, ids, scale=1.0):
    """``scale * table[ids]``: table (n, k) float32 / bfloat16 / float16, ids int32 / int64 of any shape ->
    ids.shape + (k,) in the table's type, rounded once. An id outside [0, n) (-1) gives a row of zeros.
    Differentiable in table (:func:`lookup_grad`)."""
    torch = _t()
    if torch.is_grad_enabled() and getattr(table, "requires_grad", False):
        return _function("lookup").apply(table, ids, scale)
    return _lookup(table, ids, scale)


def _lookup(table, ids, scale):
    torch = _t()
    ld = _rows(table, "table", tuple(_TYPES))
    if table.shape[0] < 1:
        raise ValueError("the table must have at least one row")
    wide = _ids(ids, "ids", table.device)
    n, k = ids.numel(), table.shape[1]
    out = torch.empty(tuple(ids.shape) + (k,), dtype=table.dtype, device=table.device)
    check(lib().blp_lookup(table.device.index, _stream(table.device), _TYPES[table.dtype], table.data_ptr(), ld,
                           table.shape[0], k, ids.data_ptr(), wide, n, _scale(scale), out.data_ptr(), k))
    return out


def lookup_grad(grad, ids, n_rows, scale=1.0, into=None):
    """The gradient of :func:`lookup` in its table: (n_rows, k) with row r = scale * the sum of grad[i] over
    ids[i] == r, in 32 bits and ascending i (the same every time), rounded to grad's type once; rows
    without ids are zero. grad: ids.shape + (k,). With `into` (n_rows, k) the sums are added to what it
    holds -- e.g. the softmax loss's gradient of the same table -- and it is returned."""
    torch = _t()
    if not isinstance(grad, torch.Tensor) or not isinstance(ids, torch.Tensor) or grad.dim() < 1 \
            or tuple(grad.shape[:-1]) != tuple(ids.shape):
        raise ValueError("grad must have the shape of ids and one more dimension")
    k, n = grad.shape[-1], ids.numel()
    if grad.dim() != 2:
        if not grad.is_contiguous():
            raise ValueError("grad must be contiguous")
        grad = grad.view(n, k)
    ld = _rows(grad, "grad", tuple(_TYPES))
    wide = _ids(ids, "ids", grad.device)
    n_rows = int(n_rows)
    if n_rows < 1:
        raise ValueError("n_rows must be at least 1")
    if into is None:
        out, ldo = torch.empty((n_rows, k), dtype=grad.dtype, device=grad.device), k
    else:
        out, ldo = into, _rows(into, "into", (grad.dtype,))
        if tuple(into.shape) != (n_rows, k) or into.device != grad.device:
            raise ValueError("into must be of shape %s on %s" % ((n_rows, k), grad.device))
    b = ctypes.c_int64(0)
    check(lib().blp_lookup_grad_workspace(_TYPES[grad.dtype], n, n_rows, k, ctypes.byref(b)))
    ws = torch.empty(b.value, dtype=torch.uint8, device=grad.device)
    check(lib().blp_lookup_grad(grad.device.index, _stream(grad.device), _TYPES[grad.dtype], grad.data_ptr(), ld,
                                ids.data_ptr(), wide, n, n_rows, k, _scale(scale), out.data_ptr(), ldo,
                                0 if into is None else 1, ws.data_ptr(), ws.numel()))
    return out


def quantize_rows(x):
    """-> (q int8 (n, k), s float32 (n,)): s = max|x| / 127 of each row, q = x / s rounded to the nearest whole
    number (halves to the even one). A row of zeros has s = 0; a row with a NaN or an infinity s = NaN.
    The rows of q are padded to multiples of 16 bytes (its stride), as :func:`int8_scores` likes them."""
    torch = _t()
    ld = _rows(x, "x", tuple(_TYPES))
    n, k = x.shape
    q = torch.empty((n, (k + 15) // 16 * 16), dtype=torch.int8, device=x.device)
    s = torch.empty((n,), dtype=torch.float32, device=x.device)
    check(lib().blp_quantize_rows(x.device.index, _stream(x.device), _TYPES[x.dtype], x.data_ptr(), ld, n, k, q.data_ptr(),
                                  q.shape[1], s.data_ptr()))
    return q[:, :k], s


def int8_scores(q, s, table_q, table_s, dtype=None):
    """``s[:, None] * table_s * (q @ table_q.T)``: every score of the catalogue from 8-bit factors and their row
    scales (:func:`quantize_rows`). q (m, k), table_q (n, k) int8, k < 131072; s (m,), table_s (n,) float32.
    The products are summed exactly in 32-bit integers; scaled in float32 and rounded once to `dtype`
    (float32, the default, bfloat16 or float16)."""
    torch = _t()
    dtype = torch.float32 if dtype is None else dtype
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, bfloat16 or float16 (got %s)" % (dtype,))
    ldq, ldt = _rows(q, "q", (torch.int8,)), _rows(table_q, "table_q", (torch.int8,))
    m, k = q.shape
    n = table_q.shape[0]
    if table_q.shape[1] != k or table_q.device != q.device:
        raise ValueError("q %s and table_q %s must have rows of the same length on one device" % (
            tuple(q.shape), tuple(table_q.shape)))
    if k >= 1 << 17:
        raise ValueError("k must be below 131072: longer sums do not fit 32 bits")
    if n < 1:
        raise ValueError("the catalogue must have at least one row")
    for t, what, rows in ((s, "s", m), (table_s, "table_s", n)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != q.device or tuple(t.shape) != (rows,) \
                or not t.is_contiguous():
            raise ValueError("%s must be a contiguous float32 tensor of shape (%d,) on %s" % (what, rows, q.device))
    out = torch.empty((m, n), dtype=dtype, device=q.device)
    b = ctypes.c_int64(0)
    check(lib().blp_scores8_workspace(q.data_ptr(), ldq, table_q.data_ptr(), ldt, m, n, k, ctypes.byref(b)))
    ws = torch.empty(b.value, dtype=torch.uint8, device=q.device)
    check(lib().blp_scores8(q.device.index, _stream(q.device), q.data_ptr(), ldq, s.data_ptr(), table_q.data_ptr(), ldt,
                            table_s.data_ptr(), m, n, k, _TYPES[dtype], out.data_ptr(), n, ws.data_ptr(), ws.numel()))
    return out


_fn = {}


def _function(which):
    """The autograd functions, made on first use (torch is imported lazily)."""
    if not _fn:
        torch = _t()

        class SoftmaxLoss(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, table, target, scale, reduction):
                out, lse, total, _, _ = _loss_forward(x, table, target, scale, reduction, False)
                ctx.save_for_backward(x, table, target, lse, total)
                ctx.scale, ctx.reduction = scale, reduction
                return out.clone()

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, grad):
                x, table, target, lse, total = ctx.saved_tensors
                count = total[1] if ctx.reduction == "mean" else None
                dx, dt = softmax_loss_backward(grad.contiguous(), lse, count, x, table, target, ctx.scale,
                                               ctx.needs_input_grad[0], ctx.needs_input_grad[1])
                return dx, dt, None, None, None

        class Lookup(torch.autograd.Function):
            @staticmethod
            def forward(ctx, table, ids, scale):
                ctx.save_for_backward(ids)
                ctx.scale, ctx.n_rows = scale, table.shape[0]
                return _lookup(table, ids, scale)

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, grad):
                (ids,) = ctx.saved_tensors
                return lookup_grad(grad.contiguous(), ids, ctx.n_rows, ctx.scale), None, None

        _fn.update(loss=SoftmaxLoss, lookup=Lookup)
    return _fn[which]
