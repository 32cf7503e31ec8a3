"""Operators of latent factors on device tensors: row lookup with its gradient (blp_lookup*), the
softmax loss over the whole catalogue with its gradients (blp_softmax_loss*), and scores of the catalogue
from 8-bit factors (blp_quantize_rows, blp_scores8) -- all in blp.h.

They stand beside :class:`blp.factor.DeviceSVD`, whose factors, copied to float32 (or halves) tensors, they read, train
and score: rows of a user table and of a business table, ``k`` components a row --
``users = torch.from_numpy(svd.us).float().cuda()``, and back ``DeviceSVD(users.double().cpu().numpy(), ...)``.

Every argument that holds data is a torch tensor on one GPU, its rows contiguous (a row stride larger than the
row is fine); the work is queued on torch's current stream of that device, workspaces come from torch's
allocator, and nothing waits for the device. Wrong arguments raise ValueError before anything is queued: row strides of the loss's operands past 2^20
elements and of 8-bit ones past 2^22 are among them.
"""
import ctypes

from . import _lib
from ._lib import BLPError, lib

_INF = float("inf")
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

class ArgumentError(BLPError, ValueError):
    """Arguments that the library refuses (BLP_E_ARG): sizes and strides past its limits."""


def check(rc):
    if rc == -1:
        raise ArgumentError(rc, lib().blp_last_error().decode(errors="replace"))
    return _lib.check(rc)


_torch = None
_forward_ad = None
_TYPES = {}   # torch dtype -> BLP_F32 / BLP_BF16 / BLP_F16
_INT8 = {}
_stream = None


def _t():
    """torch, imported on the first call: the graph engine works without it."""
    global _torch, _forward_ad, _stream
    if _torch is None:
        import torch
        from torch.autograd import forward_ad as _forward_ad

        _TYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        _INT8[torch.int8] = 3
        # the current stream's handle on a device index; the public accessor makes two objects on the way
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _torch = torch
    return _torch


def _say(t):
    return "%s %s on %s" % (tuple(t.shape), t.dtype, t.device) if isinstance(t, _torch.Tensor) else str(type(t))


def _plain(t, what):
    """Refuse what the kernels, which see a tensor's memory alone, would answer wrongly without an error. A dual tensor
    of forward-mode differentiation: a result without a tangent would be a derivative of zero (outside of a level there
    are none: that is all the common path looks at). A traced one: the trace would hold the allocation of the outputs and nothing that fills
    them (any tensor's sizes are numbers, but tensors while torch.jit traces; _rows looks)."""
    if getattr(_forward_ad, "_current_level", 0) >= 0 and isinstance(t, _torch.Tensor) \
            and _forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError("%s: forward-mode derivatives are not implemented" % what)


def _positive(t, what):
    """Refuse a negated view (z.conj().imag), whose memory holds the values before the sign. Its elements are two apart: only
    one of single elements passes for contiguous."""
    if t.is_neg():
        raise ValueError("%s must not be a negated view (resolve_neg() makes a tensor of it)" % what)


def _rows(t, what, dtypes):
    """The row stride of `t`, checked to be (n, k) rows: a 2-d tensor on a GPU whose rows are contiguous and do not
    overlap."""
    _plain(t, what)
    if isinstance(t, _torch.Tensor) and t.dim() == 2:
        n, k = t.shape
        if type(n) is not int:
            raise RuntimeError("%s: this call cannot be traced" % what)
        if t.dtype in dtypes and t.is_cuda:
            ld, step = t.stride()
            if k < 1 or (k > 1 and step != 1) or (n > 1 and ld < k):
                raise ValueError("%s must have contiguous, non-overlapping rows of at least one element (shape %s, strides %s)" % (
                    what, (n, k), (ld, step)))
            if k == 1:
                _positive(t, what)
            return ld if n > 1 else k
    raise ValueError("%s must be a 2-d GPU tensor of %s (got %s)" % (what, " / ".join(str(d)[6:] for d in dtypes), _say(t)))


def _ids(t, what, device, n=None):
    """1 for int64, 0 for int32 ids: a contiguous tensor on `device`, of shape (n,) where n is given."""
    wide = isinstance(t, _torch.Tensor) and (1 if t.dtype == _torch.int64 else 0 if t.dtype == _torch.int32 else None)
    if wide is None or wide is False or t.device != device or not t.is_contiguous() or (n is not None and t.shape != (n,)):
        raise ValueError("%s must be a contiguous int32 / int64 tensor%s on %s (got %s)" % (
            what, "" if n is None else " of shape (%d,)" % n, device, _say(t)))
    return wide


def _floats(t, what, device, shapes):
    _plain(t, what)
    if not (isinstance(t, _torch.Tensor) and t.dtype == _torch.float32 and t.device == device and t.is_contiguous()
            and t.shape in shapes):
        raise ValueError("%s must be a contiguous float32 tensor of shape %s on %s (got %s)" % (
            what, " or ".join(str(tuple(x)) for x in shapes), device, _say(t)))
    if t.numel() == 1:
        _positive(t, what)


def _bytes(like, n):
    return like.new_empty(n, dtype=_torch.uint8)


_REDUCTIONS = ("mean", "sum", "none")


def _loss_args(x, table, target, scale, reduction):
    _t()
    scale = _scale(scale)
    ldx = _rows(x, "x", _TYPES)
    if not isinstance(table, _torch.Tensor) or table.dtype != x.dtype:
        raise ValueError("x and table must be tensors of the same type (got %s and %s)" % (_say(x), _say(table)))
    ldt = _rows(table, "table", _TYPES)
    if table.shape[1] != x.shape[1] or table.device != x.device:
        raise ValueError("x %s and table %s must have rows of the same length on one device" % (
            tuple(x.shape), tuple(table.shape)))
    if table.shape[0] < 1:
        raise ValueError("the catalogue must have at least one row")
    wide = _ids(target, "target", x.device, x.shape[0])
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be one of %s (got %r)" % (", ".join(_REDUCTIONS), reduction))
    return ldx, ldt, wide, scale


def _loss_workspace(x, ldx, table, ldt, forward, grads):
    n = ctypes.c_int64(0)
    m, k = x.shape
    check(lib().blp_softmax_loss_workspace(_TYPES[x.dtype], x.data_ptr(), ldx, table.data_ptr(), ldt, m, table.shape[0], k,
                                           forward, grads, ctypes.byref(n)))
    return n.value


def _loss_forward(x, table, target, scale, reduction, grads, keep=False):
    """-> (loss or total, lse, total, dx, dtable); lse and total only where asked to `keep` them"""
    ldx, ldt, wide, scale = _loss_args(x, table, target, scale, reduction)
    m, k = x.shape
    device = x.device
    need = _loss_workspace(x, ldx, table, ldt, 1, grads)
    summed = reduction != "none"
    # what the caller does not get lies behind the workspace: the rows' lse, and their losses where they are summed up
    ws = _bytes(x, need + 8 * m)
    tail = ws.data_ptr() + need
    lse = x.new_empty(m, dtype=_torch.float32) if keep else None
    total = x.new_empty(2, dtype=_torch.float32) if summed else None
    loss = None if summed else x.new_empty(m, dtype=_torch.float32)
    dx = dt = None
    if grads:
        dx, dt = x.new_empty(m, k), x.new_empty(table.shape[0], k)
    check(lib().blp_softmax_loss(
        device.index, _stream(device.index), _TYPES[x.dtype], x.data_ptr(), ldx, table.data_ptr(), ldt, target.data_ptr(), wide,
        m, table.shape[0], k, scale, tail + 4 * m if summed else loss.data_ptr(), lse.data_ptr() if keep else tail,
        total.data_ptr() if summed else None, 1 if reduction == "mean" else 0, grads, dx.data_ptr() if grads else None, k,
        dt.data_ptr() if grads else None, k, ws.data_ptr(), need))
    return (total[0] if summed else loss), lse, total, dx, dt


def softmax_loss(x, table, target, scale=1.0, reduction="mean"):
    """Softmax cross entropy of ``scale * x @ table.T`` against ``target``, without keeping the scores.

    x (m, k), table (n, k): float32, bfloat16 or float16, the same type; target (m,) int32 / int64: the
    row of `table` that belongs to each row of x. A target outside [0, n) (-1, as in the top-k lists'
    missing slots) ignores its row: loss 0, gradient 0, whatever x holds there. reduction "mean" (over
    the rows not ignored; 0 if there is none), "sum" or "none" (one loss a row). Returns float32;
    differentiable in x and table (not inside a graph capture: capture :func:`softmax_loss_grad`).
    Sums and the softmax's statistics are held in 32 bits, and gradients are rounded to the type once: the
    softmax's differences that they sum are held as two halves each, to 2^-16 (bfloat16) or 2^-22 (float16).
    Float32 factors are multiplied as sums of three bfloat16 each, with 32-bit results; they have to be finite."""
    torch = _t()
    if torch.is_grad_enabled() and (getattr(x, "requires_grad", False) or getattr(table, "requires_grad", False)):
        return _function("loss").apply(x, table, target, _scale(scale), reduction)
    return _loss_forward(x, table, target, scale, reduction, 0)[0]


def softmax_loss_grad(x, table, target, scale=1.0, reduction="mean"):
    """-> (loss, dx, dtable): :func:`softmax_loss` ("mean" or "sum") and its gradients in one call, for
    training loops that do not go through autograd."""
    if reduction == "none":
        raise ValueError("softmax_loss_grad: reduction must be mean or sum")
    loss, _, _, dx, dt = _loss_forward(x, table, target, scale, reduction, 1)
    return loss, dx, dt


def softmax_loss_forward(x, table, target, scale=1.0, reduction="mean"):
    """-> (loss, lse, count): :func:`softmax_loss` and what :func:`softmax_loss_backward` takes of it, for loops that do not go
    through autograd: lse (m,) float32, each row's log-sum-exp (of a row that is ignored: anything); count
    the number of rows not ignored (at least 1; float32) for "mean", else None."""
    loss, lse, total, _, _ = _loss_forward(x, table, target, scale, reduction, 0, keep=True)
    return loss, lse, total[1] if reduction == "mean" else None


def softmax_loss_backward(grad, lse, count, x, table, target, scale=1.0, need_x=True, need_table=True):
    """-> (dx, dtable) of :func:`softmax_loss`: `grad` float32, one value or one a row; `lse` (m,) and `count`,
    which divides the gradient (mean) or is None, from :func:`softmax_loss_forward`."""
    ldx, ldt, wide, scale = _loss_args(x, table, target, scale, "none")
    m, k = x.shape
    device = x.device
    _floats(grad, "grad", device, ((), (1,), (m,)))
    _floats(lse, "lse", device, ((m,),))
    if count is not None:
        _floats(count, "count", device, ((), (1,)))
    dx = x.new_empty(m, k) if need_x else None
    dt = x.new_empty(table.shape[0], k) if need_table else None
    ws = _bytes(x, _loss_workspace(x, ldx, table, ldt, 0, 1))
    check(lib().blp_softmax_loss_backward(
        device.index, _stream(device.index), _TYPES[x.dtype], x.data_ptr(), ldx, table.data_ptr(), ldt, target.data_ptr(), wide,
        m, table.shape[0], k, scale, lse.data_ptr(), grad.data_ptr(), 1 if grad.numel() > 1 else 0,
        None if count is None else count.data_ptr(), None if dx is None else dx.data_ptr(), k,
        None if dt is None else dt.data_ptr(), k, ws.data_ptr(), ws.numel()))
    return dx, dt


def _scale(scale):
    """The number; a tensor of one element is one if nothing would be lost: neither its derivative nor its place in a trace."""
    if type(scale) is not float and isinstance(scale, _torch.Tensor):
        _plain(scale, "scale")
        if scale.requires_grad and _torch.is_grad_enabled():
            raise ValueError("scale must not require a gradient: its derivative is not taken")
        if _torch.jit.is_tracing():
            raise RuntimeError("scale: this call cannot be traced")
    scale = float(scale)
    if not abs(scale) < _INF:
        raise ValueError("scale must be finite (got %r)" % scale)
    return scale


def lookup(table, ids, scale=1.0):
    """``scale * table[ids]``: table (n, k) float32 / bfloat16 / float16, ids int32 / int64 of any shape ->
    ids.shape + (k,) in the table's type, rounded once. An id outside [0, n) (-1) gives a row of zeros.
    Differentiable in table (not inside a graph capture: capture :func:`lookup_grad`)."""
    torch = _t()
    if torch.is_grad_enabled() and getattr(table, "requires_grad", False):
        return _function("lookup").apply(table, ids, _scale(scale))
    return _lookup(table, ids, scale)


def _lookup(table, ids, scale):
    _t()
    scale = _scale(scale)
    ld = _rows(table, "table", _TYPES)
    rows, k = table.shape
    if rows < 1:
        raise ValueError("the table must have at least one row")
    device = table.device
    wide = _ids(ids, "ids", device)
    out = table.new_empty(*ids.shape, k)
    check(lib().blp_lookup(device.index, _stream(device.index), _TYPES[table.dtype], table.data_ptr(), ld, rows, k,
                           ids.data_ptr(), wide, ids.numel(), scale, out.data_ptr(), k))
    return out


def lookup_grad(grad, ids, n_rows, scale=1.0, into=None):
    """The gradient of :func:`lookup` in its table: (n_rows, k) with row r = scale * the sum of grad[i] over
    ids[i] == r, rounded to grad's type once: up to 64 entries at a time in 32 bits and ascending i, these sums
    in 64 bits and a fixed order (the same every time); rows without ids are zero. grad: ids.shape + (k,). With
    `into` (n_rows, k) the sums are added to what it holds -- e.g. the softmax loss's gradient of the same table -- and it is returned; to autograd that is a change
    in place, and `into` must not require a gradient (but under torch.no_grad)."""
    torch = _t()
    scale = _scale(scale)
    if not isinstance(grad, torch.Tensor) or not isinstance(ids, torch.Tensor) or grad.dim() < 1 \
            or tuple(grad.shape[:-1]) != tuple(ids.shape):
        raise ValueError("grad must have the shape of ids and one more dimension")
    k, n = grad.shape[-1], ids.numel()
    if grad.dim() != 2:
        if not grad.is_contiguous():
            raise ValueError("grad must be contiguous")
        grad = grad.view(n, k)
    ld = _rows(grad, "grad", _TYPES)
    wide = _ids(ids, "ids", grad.device)
    n_rows = int(n_rows)
    if n_rows < 1:
        raise ValueError("n_rows must be at least 1")
    if into is None:
        out, ldo = grad.new_empty(n_rows, k), k
    else:
        out, ldo = into, _rows(into, "into", (grad.dtype,))
        if into.requires_grad and torch.is_grad_enabled():
            raise ValueError("into must not require a gradient: the sums are added without a record of it")
        if tuple(into.shape) != (n_rows, k) or into.device != grad.device:
            raise ValueError("into must be of shape %s on %s" % ((n_rows, k), grad.device))
        if n and into.data_ptr() < grad.data_ptr() + ((n - 1) * ld + k) * grad.element_size() \
                and grad.data_ptr() < into.data_ptr() + ((n_rows - 1) * ldo + k) * grad.element_size():
            raise ValueError("into must not overlap grad")
    b = ctypes.c_int64(0)
    check(lib().blp_lookup_grad_workspace(_TYPES[grad.dtype], n, n_rows, k, ctypes.byref(b)))
    ws = _bytes(grad, b.value)
    check(lib().blp_lookup_grad(grad.device.index, _stream(grad.device.index), _TYPES[grad.dtype], grad.data_ptr(), ld,
                                ids.data_ptr(), wide, n, n_rows, k, scale, out.data_ptr(), ldo,
                                0 if into is None else 1, ws.data_ptr(), ws.numel()))
    if into is not None:
        torch.autograd.graph.increment_version(into)  # autograd sees that what it may have kept of `into` has changed
    return out


def quantize_rows(x):
    """-> (q int8 (n, k), s float32 (n,)): s = max|x| / 127 of each row, q = x / s rounded to the nearest whole
    number (halves to the even one). A row of zeros has s = 0; a row with a NaN or an infinity s = NaN.
    The rows of q are padded to multiples of 16 bytes (its stride), as :func:`int8_scores` likes them."""
    _t()
    ld = _rows(x, "x", _TYPES)
    n, k = x.shape
    device = x.device
    kp = (k + 15) // 16 * 16
    q = x.new_empty(n, kp, dtype=_torch.int8)
    s = x.new_empty(n, dtype=_torch.float32)
    check(lib().blp_quantize_rows(device.index, _stream(device.index), _TYPES[x.dtype], x.data_ptr(), ld, n, k, q.data_ptr(),
                                  kp, s.data_ptr()))
    return (q if kp == k else q[:, :k]), s


def int8_scores(q, s, table_q, table_s, dtype=None):
    """``s[:, None] * table_s * (q @ table_q.T)``: every score of the catalogue from 8-bit factors and their row
    scales (:func:`quantize_rows`). q (m, k), table_q (n, k) int8, k < 131072; s (m,), table_s (n,) float32.
    The products are summed exactly in 32-bit integers; scaled in float32 and rounded once to `dtype`
    (float32, the default, bfloat16 or float16). Not differentiable."""
    torch = _t()
    dtype = torch.float32 if dtype is None else dtype
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, bfloat16 or float16 (got %s)" % (dtype,))
    ldq, ldt = _rows(q, "q", _INT8), _rows(table_q, "table_q", _INT8)
    m, k = q.shape
    n = table_q.shape[0]
    device = q.device
    if table_q.shape[1] != k or table_q.device != device:
        raise ValueError("q %s and table_q %s must have rows of the same length on one device" % (
            tuple(q.shape), tuple(table_q.shape)))
    if k >= 1 << 17:
        raise ValueError("k must be below 131072: longer sums do not fit 32 bits")
    if n < 1:
        raise ValueError("the catalogue must have at least one row")
    _floats(s, "s", device, ((m,),))
    _floats(table_s, "table_s", device, ((n,),))
    out = q.new_empty(m, n, dtype=dtype)
    qp, tp = q.data_ptr(), table_q.data_ptr()
    b = ctypes.c_int64(0)
    check(lib().blp_scores8_workspace(qp, ldq, tp, ldt, m, n, k, ctypes.byref(b)))
    ws = _bytes(q, b.value) if b.value else None
    check(lib().blp_scores8(device.index, _stream(device.index), qp, ldq, s.data_ptr(), tp, ldt, table_s.data_ptr(), m, n, k,
                            _TYPES[dtype], out.data_ptr(), n, ws.data_ptr() if b.value else None, b.value))
    return out


def _no_capture(what, instead):
    """Autograd ties a leaf's gradient to the stream on which the leaf was first used, and waits for that stream in the
    backward pass; inside a capture that cannot be honoured, and the process may end. The explicit calls
    queue their work on the current stream alone."""
    if _torch.cuda.is_current_stream_capturing():
        raise RuntimeError("%s: gradients through autograd cannot be captured into a graph; capture %s instead" % (what, instead))


_fn = {}


def _function(which):
    """The autograd functions, made on first use (torch is imported lazily)."""
    if not _fn:
        torch = _t()

        class SoftmaxLoss(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, table, target, scale, reduction):
                _no_capture("softmax_loss", "softmax_loss_grad")
                out, lse, total, _, _ = _loss_forward(x, table, target, scale, reduction, 0, keep=True)
                ctx.save_for_backward(x, table, target, lse, *(() if total is None else (total,)))
                ctx.scale, ctx.reduction = scale, reduction
                return out.clone()

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, grad):
                _no_capture("softmax_loss", "softmax_loss_grad")
                x, table, target, lse = ctx.saved_tensors[:4]
                count = ctx.saved_tensors[4][1] if ctx.reduction == "mean" else None
                dx, dt = softmax_loss_backward(grad.contiguous(), lse, count, x, table, target, ctx.scale,
                                               ctx.needs_input_grad[0], ctx.needs_input_grad[1])
                return dx, dt, None, None, None

        class Lookup(torch.autograd.Function):
            @staticmethod
            def forward(ctx, table, ids, scale):
                _no_capture("lookup", "lookup_grad")
                ctx.save_for_backward(ids)
                ctx.scale, ctx.n_rows = scale, table.shape[0]
                return _lookup(table, ids, scale)

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, grad):
                _no_capture("lookup", "lookup_grad")
                (ids,) = ctx.saved_tensors
                return lookup_grad(grad.contiguous(), ids, ctx.n_rows, ctx.scale), None, None

        _fn.update(loss=SoftmaxLoss, lookup=Lookup)
    return _fn[which]
