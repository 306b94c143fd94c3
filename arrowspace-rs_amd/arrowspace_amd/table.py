"""Operators over a table of rows (what an index holds), over the C ABI: softmax cross entropy against all its items with the
gradient, and products with a table held in 4 bits.  They have no counterpart in the reference.

Matrices are torch tensors (on a GPU: used in place, on torch's current stream of that GPU, capturable into a graph) or numpy arrays
(staged; results come back as numpy arrays, complete).  Results lie where the first argument does; the others may be host memory or on
one GPU, and as soon as one of them is, the call runs on torch's current stream there.  The host waits for the GPU only where host memory
is copied, and where a thread goes on to another stream than its last call's: for that call's stream.  Rows may be rows of a wider
tensor; the values of a row must be adjacent.  Tensors that require gradients get them: cross_entropy is differentiable (once), and a
backward pass through the scores of a Table4, which have no gradient, raises.
"""
import ctypes as C
import threading

import numpy as np

from . import _lib
from ._lib import ArrowSpaceError, AS_BF16, AS_F16, AS_F32, AS_F64, is_tensor
from .api import Context, DeviceArray

_DTYPES = {"float64": AS_F64, "float32": AS_F32, "bfloat16": AS_BF16, "float16": AS_F16}
_NAMES = {AS_F64: "float64", AS_F32: "float32", AS_BF16: "bfloat16", AS_F16: "float16"}
_local = threading.local()
_torch = None          # the module, once a tensor has been seen
_raw_stream = None     # device index -> address of torch's current stream there
_kinds, _types = {}, {}  # torch dtype -> name and back
_Loss = _Scores = None  # torch.autograd.Functions


def _need_torch():
    global _torch, _raw_stream
    import torch
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    for name in ("float64", "float32", "bfloat16", "float16", "int64", "uint8"):
        _types[name] = getattr(torch, name)
        _kinds[_types[name]] = name
    _torch = torch
    _differentiable()


def _differentiable():
    """The operators as torch.autograd.Functions (made once torch is there)."""
    global _Loss, _Scores
    once = _torch.autograd.function.once_differentiable

    class Loss(_torch.autograd.Function):
        @staticmethod
        def forward(node, x, table, bias, targets, scale, ignore_index, ctx):
            losses, lse = _cross_entropy(x, table, targets, bias, scale, ignore_index, ctx)
            kept = [x, table, bias, targets, lse]
            # (host arrays beside tensors: on the node itself)
            node.save_for_backward(*[a if a is None or isinstance(a, _torch.Tensor) else None for a in kept])
            node.host = [None if a is None or isinstance(a, _torch.Tensor) else a for a in kept]
            node.scale, node.ignore_index = scale, ignore_index
            node.set_materialize_grads(False)
            return losses, lse

        @staticmethod
        @once
        def backward(node, grad_losses, grad_lse):
            none = (None,) * 7
            if grad_losses is None and grad_lse is None:
                return none
            x, table, bias, targets, lse = [h if t is None else t for t, h in zip(node.saved_tensors, node.host)]
            if grad_losses is None:
                grad_losses = _torch.zeros_like(lse)
            need = node.needs_input_grad
            # (on the thread that runs this, with a context of its own: the forward call's is its caller's)
            grads = cross_entropy_backward(x, table, targets, lse, grad_losses, bias=bias, scale=node.scale, ignore_index=node.ignore_index,
                                           grad_lse=grad_lse, need_x=need[0], need_table=need[1], need_bias=need[2])
            return tuple(g if g is None else g.to(a.device) for g, a in zip(grads, (x, table, bias))) + none[3:]

    class Scores(_torch.autograd.Function):
        @staticmethod
        def forward(node, x, table, ctx):
            return table._scores(x, ctx)

        @staticmethod
        def backward(node, grad):
            raise ArrowSpaceError(_lib.AS_ERR_UNSUPPORTED, "the scores of a table in 4 bits have no gradient")

    _Loss, _Scores = Loss, Scores


def _recording():
    """Whether torch records calls for a backward pass."""
    if _torch is None:
        _need_torch()
    return _torch.is_grad_enabled()


def _requires_grad(a):
    return getattr(a, "requires_grad", False)


def _thread_context(device):
    """The calling thread's own context on a device (a context is not re-entrant)."""
    table = getattr(_local, "contexts", None)
    if table is None:
        table = _local.contexts = {}
    ctx = table.get(device)
    if ctx is None:
        before = _torch.cuda.current_device() if _torch is not None and _torch.cuda.is_available() else None
        ctx = table[device] = Context(device)
        if before is not None and before != device:
            _torch.cuda.set_device(before)
    return ctx


class _Call:
    """Where a call's data live, and its context with the right stream: torch's current one of the GPU that ANY of the arguments is on
    (that is where the others are written too, whether the first one is host memory or not).  Outputs lie beside the first."""
    __slots__ = ("device", "cuda", "ctx", "torch")

    def __init__(self, first, ctx, others=()):
        self.device, self.cuda, self.torch = None, False, False
        index = None
        if is_tensor(first):
            if _torch is None:
                _need_torch()
            self.torch = True
            self.device = first.device
            self.cuda = first.is_cuda
        if self.cuda:
            index = self.device.index   # (a tensor of another device than this one's is refused by the library)
        else:
            for a in others:
                if a is not None and is_tensor(a) and a.is_cuda:
                    if _torch is None:
                        _need_torch()
                    index = a.device.index
                    break
        if index is not None:
            if ctx is None:
                ctx = _thread_context(index)
            elif ctx.device != index:
                raise ArrowSpaceError(_lib.AS_ERR_ARG, "tensors of device %d, a context of device %d" % (index, ctx.device))
            st = _raw_stream(index)
            if getattr(ctx, "_stream", "own") != st:
                ctx.set_stream(st)
        elif ctx is None:
            ctx = _thread_context(0)
        self.ctx = ctx

    def empty(self, shape, dtype):
        """(array, address) of an output beside the call's inputs; dtype a name."""
        if self.torch:
            a = _torch.empty(shape, dtype=_types[dtype], device=self.device)
            return a, a.data_ptr()
        a = np.empty(shape, dtype=dtype)
        return a, a.ctypes.data

    def workspace(self, size):
        """(tensor, address, bytes): torch's own allocator on a GPU, so that a captured graph keeps what it uses; else the library's."""
        if not size or not self.cuda:
            return None, None, 0
        w = _torch.empty(size, dtype=_torch.uint8, device=self.device)
        return w, w.data_ptr(), size


def _name(a):
    name = _kinds.get(a.dtype)
    return name if name is not None else str(a.dtype).replace("torch.", "")


def _known(a, what):
    if isinstance(a, DeviceArray):
        raise TypeError("%s is a DeviceArray, which is not taken here: torch tensors or numpy arrays" % what)


def _matrix(a, what):
    """(array, rows, columns, row stride in elements, address) of a matrix whose rows' values are adjacent."""
    if not is_tensor(a):
        a = np.asarray(a)
        if a.ndim != 2:
            raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "%s must be a matrix, got %d dimensions" % (what, a.ndim))
        a = np.ascontiguousarray(a)
        return a, a.shape[0], a.shape[1], a.shape[1], a.ctypes.data
    _known(a, what)
    if a.dim() != 2:
        raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "%s must be a matrix, got %d dimensions" % (what, a.dim()))
    n, d = a.shape
    step, inner = a.stride()
    if d > 1 and inner != 1:
        raise ArrowSpaceError(_lib.AS_ERR_ARG, "the values of a row of %s must be adjacent" % what)
    if n <= 1:
        step = max(step, d)
    if step < d:
        raise ArrowSpaceError(_lib.AS_ERR_ARG, "rows of %s overlap" % what)
    return a, n, d, step, a.data_ptr()


def _vector(a, n, dtype, what):
    """Address of a dense vector of n elements, and the array that has to stay alive."""
    if a is None:
        return None, None
    if not is_tensor(a):
        a = np.asarray(a)
        if a.dtype != np.dtype(dtype):
            raise TypeError("%s must be %s, got %s" % (what, dtype, a.dtype))
        a = np.ascontiguousarray(a)
        if a.shape != (n,):
            raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "%s must have %d elements, has shape %s" % (what, n, a.shape))
        return a.ctypes.data, a
    _known(a, what)
    if _name(a) != dtype:
        raise TypeError("%s must be %s, got %s" % (what, dtype, a.dtype))
    if tuple(a.shape) != (n,):
        raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "%s must have %d elements, has shape %s" % (what, n, tuple(a.shape)))
    a = a.contiguous()   # (an expanded gradient, say)
    return a.data_ptr(), a


def _loss_args(x, table, bias, targets, ctx, *others):
    first = x
    x, n, d, xs, xp = _matrix(x, "x")
    table, v, dw, ts, tp = _matrix(table, "table")
    if d != dw:
        raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "rows of %d values against a table of %d" % (d, dw))
    kind = _DTYPES.get(_name(x))
    if kind is None or kind == AS_F64 or _name(table) != _name(x):
        raise TypeError("x and table must both be float32, bfloat16 or float16, got %s and %s" % (x.dtype, table.dtype))
    bp, bias = _vector(bias, v, "float32", "bias")
    yp, targets = _vector(targets, n, "int64", "targets")
    if yp is None:
        raise ArrowSpaceError(_lib.AS_ERR_ARG, "null argument")
    call = _Call(first, ctx, (table, bias, targets) + others)
    return call, (xp, n, xs, tp, v, ts, d, kind, bp, yp), (x, table, bias, targets)


def cross_entropy(x, table, targets, bias=None, scale=1.0, ignore_index=-100, ctx=None):
    """Softmax cross entropy of every row of x (n x d) against all rows of the table (v x d), the n x v logits never kept:
    (losses, lse), both float32 of n.  logits = scale * x @ table.T + bias; losses are 0 where targets == ignore_index and where the
    bias (-inf) leaves no item.  The mean over the counted rows is losses.sum() / count.  Tensors: x, table and bias have gradients,
    through both results; scale is a number."""
    try:
        graph = x.requires_grad or table.requires_grad or (bias is not None and bias.requires_grad) or (type(scale) is not float and _requires_grad(scale))
    except AttributeError:   # (host arrays)
        graph = any(map(_requires_grad, (x, table, bias, scale)))
    if graph and is_tensor(x) and _recording():
        if is_tensor(scale):
            raise TypeError("scale is a number: it has no gradient here")
        return _Loss.apply(x, table, bias, targets, scale, ignore_index, ctx)
    return _cross_entropy(x, table, targets, bias, scale, ignore_index, ctx)


def _cross_entropy(x, table, targets, bias, scale, ignore_index, ctx):
    call, (xp, n, xs, tp, v, ts, d, kind, bp, yp), alive = _loss_args(x, table, bias, targets, ctx)
    (losses, op), (lse, lp) = call.empty((n,), "float32"), call.empty((n,), "float32")
    c = call.ctx
    lib = c.lib
    ws, wp, wb = call.workspace(lib.as_cross_entropy_workspace(n, v, d, kind, 0))
    rc = lib.as_cross_entropy(c.h, xp, n, xs, tp, v, ts, d, kind, bp, yp, int(ignore_index), float(scale), op, lp, wp, wb)
    if rc:
        c.check(rc)
    return losses, lse


def cross_entropy_backward(x, table, targets, lse, grad_losses, bias=None, scale=1.0, ignore_index=-100, grad_lse=None, need_x=True,
                           need_table=True, need_bias=True, ctx=None):
    """The gradients of cross_entropy's inputs, (grad_x, grad_table, grad_bias), from the gradients of its two outputs (grad_lse
    None: zero) and the lse that it returned.  grad_x and grad_table have the inputs' type, grad_bias is float32; None where not needed
    or where there is no bias."""
    rows = tuple(x.shape)[0]
    lp, lse = _vector(lse, rows, "float32", "lse")
    gp, grad_losses = _vector(grad_losses, rows, "float32", "grad_losses")
    ep, grad_lse = _vector(grad_lse, rows, "float32", "grad_lse")
    if lp is None or gp is None:
        raise ArrowSpaceError(_lib.AS_ERR_ARG, "null argument")
    call, (xp, n, xs, tp, v, ts, d, kind, bp, yp), alive = _loss_args(x, table, bias, targets, ctx, lse, grad_losses, grad_lse)
    none = (None, None)
    gx, gxp = call.empty((n, d), _NAMES[kind]) if need_x else none
    gw, gwp = call.empty((v, d), _NAMES[kind]) if need_table else none
    gb, gbp = call.empty((v,), "float32") if need_bias and bp is not None else none
    c = call.ctx
    lib = c.lib
    ws, wp, wb = call.workspace(lib.as_cross_entropy_workspace(n, v, d, kind, 1))
    rc = lib.as_cross_entropy_backward(c.h, xp, n, xs, tp, v, ts, d, kind, bp, yp, int(ignore_index), float(scale), lp, gp, ep, gxp, d, gwp, d,
                                       gbp, wp, wb)
    if rc:
        c.check(rc)
    return gx, gw, gb


class Table4:
    """A table of rows in 4 bits with group scales, laid out for the kernels: W = scale * (code - zero), zero 8 unless given.
    Make one from rows (pack) or from codes that exist already (from_codes); scores(x) is x @ W.T."""

    def __init__(self, ctx, handle):
        self.ctx, self.h = ctx, handle
        lib = ctx.lib
        self.n_items, self.dim, self.group = int(lib.as_table4_items(handle)), int(lib.as_table4_dim(handle)), int(lib.as_table4_group(handle))
        self.scale_dtype = _NAMES[lib.as_table4_scale_dtype(handle)]

    @classmethod
    def pack(cls, rows, group=64, scale_dtype="bfloat16", ctx=None):
        """Quantises rows (float64, float32, bfloat16 or float16): per group the largest magnitude / 7 becomes the scale."""
        first = rows
        rows, n, d, step, p = _matrix(rows, "rows")
        kind, scale_kind = _DTYPES.get(_name(rows)), _scale_kind(scale_dtype)
        if kind is None:
            raise TypeError("rows must be floating-point, got %s" % rows.dtype)
        _check_group(group)
        call = _Call(first, ctx)
        h = C.c_void_p()
        call.ctx.check(call.ctx.lib.as_table4_pack(call.ctx.h, p, n, step, d, kind, int(group), scale_kind, C.byref(h)))
        return cls(call.ctx, h)

    @classmethod
    def from_codes(cls, codes, scales, zeros=None, dim=None, group=64, ctx=None):
        """codes: uint8, n x ceil(dim / 2), column 2 j in the low half of byte j; scales: n x ceil(dim / group), float32, bfloat16 or
        float16; zeros: uint8 of the scales' shape, or None."""
        first = codes
        _check_group(group)
        codes, n, half, step, cp = _matrix(codes, "codes")
        dim = 2 * half if dim is None else int(dim)
        if _name(codes) != "uint8" or (zeros is not None and _name(zeros) != "uint8"):
            raise TypeError("codes and zeros must be uint8")
        if (dim + 1) // 2 != half:
            raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "%d columns take %d bytes a row, codes have %d" % (dim, (dim + 1) // 2, half))
        scales, sn, sg, sstep, sp = _matrix(scales, "scales")
        groups = (dim + int(group) - 1) // int(group)
        if (sn, sg) != (n, groups):
            raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "scales must be %d x %d, are %d x %d" % (n, groups, sn, sg))
        zp = None
        if zeros is not None:
            zeros, zn, zg, zstep, zp = _matrix(zeros, "zeros")
            if (zn, zg) != (n, groups):
                raise ArrowSpaceError(_lib.AS_ERR_SHAPE, "zeros must be %d x %d, are %d x %d" % (n, groups, zn, zg))
        if n > 1 and (step != half or sstep != groups or (zeros is not None and zstep != groups)):
            raise ArrowSpaceError(_lib.AS_ERR_ARG, "codes, scales and zeros must be dense")
        scale_kind = _scale_kind(_name(scales))
        call = _Call(first, ctx, (scales, zeros))
        h = C.c_void_p()
        call.ctx.check(call.ctx.lib.as_table4_import(call.ctx.h, cp, sp, zp, n, dim, int(group), scale_kind, C.byref(h)))
        return cls(call.ctx, h)

    def to_codes(self):
        """(codes, scales, zeros) as host arrays; bfloat16 scales come back as float32."""
        groups = (self.dim + self.group - 1) // self.group
        codes = np.empty((self.n_items, (self.dim + 1) // 2), dtype=np.uint8)
        zeros = np.empty((self.n_items, groups), dtype=np.uint8)
        raw = np.empty((self.n_items, groups), dtype=np.uint16 if self.scale_dtype == "bfloat16" else self.scale_dtype)
        c = _thread_context(self.ctx.device)
        c.check(c.lib.as_table4_export(c.h, self.h, codes.ctypes.data, raw.ctypes.data, zeros.ctypes.data))
        scales = (raw.astype(np.uint32) << 16).view(np.float32) if self.scale_dtype == "bfloat16" else raw
        return codes, scales, zeros

    def scores(self, x, ctx=None):
        """x @ W.T for one row or a few (float32, bfloat16 or float16), in x's type.  They have no gradient: a backward pass raises."""
        return _Scores.apply(x, self, ctx) if _requires_grad(x) and _recording() else self._scores(x, ctx)

    def _scores(self, x, ctx):
        first = x
        single = len(x.shape) == 1
        if single:
            _known(x, "x")
            x = x.reshape(1, -1)
        x, m, d, step, p = _matrix(x, "x")
        if d != self.dim:
            raise ArrowSpaceError(_lib.AS_ERR_DIM, "rows of %d values against a table of %d" % (d, self.dim))
        kind = _DTYPES.get(_name(x))
        if kind is None or kind == AS_F64:
            raise TypeError("x must be float32, bfloat16 or float16, got %s" % x.dtype)
        call = _Call(first, ctx)
        out, op = call.empty((m, self.n_items), _NAMES[kind])
        c = call.ctx
        lib = c.lib
        ws, wp, wb = call.workspace(lib.as_table4_workspace(self.h, m, kind))
        rc = lib.as_table4_scores(c.h, self.h, p, m, step, kind, op, self.n_items, wp, wb)
        if rc:
            c.check(rc)
        return out[0] if single else out

    def __del__(self):
        try:
            if self.h:
                self.ctx.lib.as_table4_destroy(self.h)
                self.h = None
        except Exception:  # noqa: BLE001 -- interpreter shutdown
            pass


def _check_group(group):
    if int(group) not in (32, 64, 128):
        raise ArrowSpaceError(_lib.AS_ERR_UNSUPPORTED, "groups of 32, 64 or 128 columns, not %d" % int(group))


def _scale_kind(name):
    kind = _DTYPES.get(str(name).replace("torch.", ""))
    if kind is None or kind == AS_F64:
        raise TypeError("scales are float32, bfloat16 or float16, not %s" % name)
    return kind
