"""Operators on a policy's logits and on gradients, for device tensors (include/connect6_amd.h part 7): what logits go through before a
move is chosen, the loss they are trained on, and the clipping of the gradients it sends back.

    y = logits_process(logits, mask=mask, bias=bias, history=moves, history_len=lens, penalties=p)
    loss, lse, total, grad = policy_loss(logits, targets, mask=mask, grad_scale=1.0 / rows)
    norm = GradClip(grads).clip(1.0)

Everything runs on torch's current stream of the tensors' device without synchronising, and can be captured into a graph.  Arguments
that do not fit raise C6Error before anything runs.  Nothing here is recorded by autograd: while it records (not under no_grad), logits, biases,
penalties, weights or upstream gradients that require a gradient are refused, and so are forward-mode duals (pass them detached; policy_loss returns
the gradient, policy_loss_grad takes the upstream one).

`import torch` comes before the first use of the library in a process that wants both on the GPU: whichever is first brings the HIP runtime
that the other then shares (torch does not start on another's)."""
import ctypes as C
import functools
import sys

import torch
import torch.autograd.forward_ad as _forward

import alphazero_connect6_amd as _pkg

from . import C6Error, Logits, _chk, lib

if _pkg._lib is not None and _pkg.device_count() > 0 and not torch.cuda.is_available():
    raise C6Error("libconnect6_amd was used before torch was imported: torch cannot share its HIP runtime; import torch first")

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INDEX = {torch.int32: 0, torch.int64: 1}
_WEIGHTS = 2
_Tensor, _F32, _I32, _U8 = torch.Tensor, torch.float32, torch.int32, torch.uint8
_written_to = torch.autograd.graph.increment_version      # tensors of the caller's that a call wrote: autograd notices where it had saved them for a backward pass


def _raw_stream(device):
    return torch.cuda.current_stream(device).cuda_stream


# the handle alone where torch has a call for it: 0.1 us instead of 1.8
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)

@functools.lru_cache(maxsize=1024)
def _loss_workspace(rows, width):
    return lib().c6_policy_loss_workspace(rows, width)


# The checks below cost a call less than its launch: messages are made when they are needed, and attributes are read once.


def _followed(t, what):
    """refuses what autograd would have to follow: the result has no record of it"""
    if t.requires_grad and torch.is_grad_enabled():
        raise C6Error(f"{what} requires a gradient: autograd does not see this operator, pass a detached tensor")
    if getattr(_forward, "_current_level", 0) >= 0 and _forward.unpack_dual(t).tangent is not None:
        raise C6Error(f"{what} carries a forward-mode tangent: autograd does not see this operator")


def _logits(x, mask):
    """-> (c6_logits, rows, width)"""
    kind = _TYPE.get(x.dtype) if isinstance(x, _Tensor) else None
    shape = x.shape if kind is not None else ()
    device = x.get_device() if kind is not None else -1
    if device < 0 or len(shape) != 2:
        raise C6Error("logits must be a [rows, width] tensor of float32, float16 or bfloat16 on the GPU")
    rows, width = shape
    if rows > 0x7fffffff or width > 1 << 30:      # (the C struct's fields would take the low 32 bits)
        raise C6Error("logits must have at most 2^31 - 1 rows of at most 2^30 entries")
    stride, step = x.stride()
    if step != 1 and width > 1:
        raise C6Error("the entries of a row of logits must lie next to each other")
    _followed(x, "the logits tensor")
    if mask is None:
        return Logits(rows, width, kind, device, x.data_ptr(), stride, None, 0, 0), rows, width
    if not isinstance(mask, _Tensor) or mask.dtype is not _U8 or mask.get_device() != device:
        raise C6Error("mask must be a uint8 tensor on the logits' device")
    shape, strides = mask.shape, mask.stride()
    if len(shape) == 1:
        shape, strides = (1, *shape), (0, *strides)
    if len(shape) != 2 or shape[1] != (width + 7) // 8 or (shape[0] != rows and shape[0] != 1):
        raise C6Error(f"mask must be [{rows}, {(width + 7) // 8}], or one row for all: one bit per entry of logits, entry v at bit v % 8 of byte v // 8")
    return Logits(rows, width, kind, device, x.data_ptr(), stride, mask.data_ptr(), 0 if shape[0] == 1 else strides[0], strides[1]), rows, width


def _written(out, x, what):
    if out is None:
        return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if not isinstance(out, _Tensor) or out.get_device() != x.get_device() or out.dtype is not x.dtype or out.shape != x.shape:
        raise C6Error(f"{what} must have the logits' shape, type and device")
    if out.requires_grad:
        raise C6Error(f"{what} must not require a gradient")
    _followed(out, what)
    if out.stride(1) != 1 and x.shape[1] > 1:
        raise C6Error(f"the entries of a row of {what} must lie next to each other")
    return out


def _rows_by(t, dtype, device, rows, width, what):
    """(pointer, row stride) of a [rows, width] / [1, width] / [width] tensor"""
    if not isinstance(t, _Tensor) or t.dtype is not dtype or t.get_device() != device:
        raise C6Error(f"{what} must be a {dtype} tensor on the logits' device")
    _followed(t, what)
    shape, stride = t.shape, t.stride()
    dim = len(shape)
    if (dim != 2 and dim != 1) or shape[-1] != width or (dim == 2 and shape[0] != rows and shape[0] != 1):
        raise C6Error(f"{what} must be [{rows}, {width}], [1, {width}] or [{width}]")
    if stride[-1] != 1 and width > 1:
        raise C6Error(f"the entries of a row of {what} must lie next to each other")
    return t.data_ptr(), 0 if dim == 1 or shape[0] == 1 else stride[0]


def _per_row(t, dtype, device, rows, what):
    if not isinstance(t, _Tensor) or t.dtype is not dtype or t.get_device() != device or t.shape != (rows,) or (rows > 1 and not t.is_contiguous()):
        raise C6Error(f"{what} must be a contiguous {dtype} tensor [{rows}] on the logits' device")
    _followed(t, what)
    return t.data_ptr()


def logits_process(logits, mask=None, bias=None, history=None, history_len=None, penalties=None, out=None):
    """Penalties for repeated moves (or tokens), a bias and a mask on logits [rows, width] (c6_logits_process):

        y = x;  if v occurs c > 0 times in the row's history:  y = (x > 0 ? x / repetition : x * repetition) - (frequency * c + presence)
        y += bias;  an entry that is not legal becomes -infinity

    mask: uint8 [rows, ceil(width / 8)], any strides (a transposed view of legal_mask's layout too), or one for all rows; set bits are legal.
    bias: float32 [width] or [rows, width].  history: int32 [rows, cap] ids (or one for all rows), of which the first history_len[r] count (int32
    [rows]; None: all); ids outside the row, such as -1, count for nothing.  penalties: float32 [3] or [rows, 3] = repetition, frequency, presence.
    out: a tensor like logits, possibly logits itself; it overlaps no other argument.  Returns out."""
    l, rows, width = _logits(logits, mask)
    dev = l.device
    given, out = out, _written(out, logits, "out")
    h = n = p = b = None
    hs = ps = bs = cap = 0
    if history is not None:
        if not isinstance(history, _Tensor) or history.dim() not in (1, 2) or penalties is None:
            raise C6Error("history must be an int32 tensor [rows, cap] or [cap], and needs penalties")
        cap = history.shape[-1]
        if cap > 1 << 30:
            raise C6Error("a row of the history has at most 2^30 ids")
        h, hs = _rows_by(history, _I32, dev, rows, cap, "history")
        p, ps = _rows_by(penalties, _F32, dev, rows, 3, "penalties")
        if history_len is not None:
            n = _per_row(history_len, _I32, dev, rows, "history_len")
    elif history_len is not None or penalties is not None:
        raise C6Error("history_len and penalties need a history")
    if bias is not None:
        b, bs = _rows_by(bias, _F32, dev, rows, width, "bias")
    _chk(lib().c6_logits_process(l, h, hs, n, cap, p, ps, b, bs, out.data_ptr(), out.stride(0), _stream(dev)))
    if given is not None:
        _written_to(out)
    return out


def _target(targets, device, rows, width):
    """-> (pointer, kind, stride)"""
    if not isinstance(targets, _Tensor) or targets.get_device() != device:
        raise C6Error("targets must be a tensor on the logits' device")
    kind = _INDEX.get(targets.dtype)
    if kind is not None:
        return _per_row(targets, targets.dtype, device, rows, "targets of indices"), kind, 0
    if targets.dtype is not _F32 or targets.dim() != 2 or targets.shape[0] != rows or targets.shape[1] != width:
        raise C6Error(f"targets must be int32 or int64 indices [{rows}], or float32 weights [{rows}, {width}]")
    _followed(targets, "targets")
    stride, step = targets.stride()
    if step != 1 and width > 1:
        raise C6Error("the weights of a row must lie next to each other")
    return targets.data_ptr(), _WEIGHTS, stride


def policy_loss(logits, targets, mask=None, grad_scale=None, grad=None):
    """Cross entropy of logits [rows, width] against targets over the legal entries (c6_policy_loss) -> (loss, lse, total), float32 [rows] each, or
    (loss, lse, total, gradient) with a grad_scale (the derivative of grad_scale * sum(loss) by the logits, in the logits' type; 1 / rows for a mean).

    targets: int32 / int64 [rows] -- the entry played; outside the row or illegal: the row adds nothing -- or float32 [rows, width] weights >= 0
    (visit counts, a teacher's distribution).  loss = sum t (lse - x), total = sum t.  mask as in logits_process.  grad: where the gradient goes,
    possibly logits itself; it overlaps no other argument.  A row with no legal entry above -infinity has loss 0, lse -infinity and gradient 0."""
    l, rows, width = _logits(logits, mask)
    dev = l.device
    t, kind, ts = _target(targets, dev, rows, width)
    g, gs, given = None, 0, grad
    if grad_scale is not None:
        grad = _written(grad, logits, "grad")
        g, gs = grad.data_ptr(), grad.stride(0)
    elif grad is not None:
        raise C6Error("grad needs a grad_scale")
    stats = torch.empty_strided((3, rows), (rows, 1), dtype=_F32, device=logits.device)
    at = stats.data_ptr()
    space, nbytes = None, _loss_workspace(rows, width)
    if nbytes:
        keep = torch.empty_strided((nbytes,), (1,), dtype=_U8, device=logits.device)
        space = keep.data_ptr()
    _chk(lib().c6_policy_loss(l, t, kind, ts, at, at + 4 * rows, at + 8 * rows, g, gs, grad_scale or 0.0, space, nbytes, _stream(dev)))
    if given is not None:
        _written_to(grad)
    loss, lse, total = stats.unbind(0)
    return (loss, lse, total) if grad is None else (loss, lse, total, grad)


def policy_loss_grad(logits, targets, lse, total, dloss, mask=None, out=None):
    """The gradient by the logits from the lse and total of policy_loss and the upstream gradient dloss, float32 [rows] or [1] (c6_policy_loss_grad).
    out: where it goes, possibly logits itself; it overlaps no other argument."""
    l, rows, width = _logits(logits, mask)
    dev = l.device
    t, kind, ts = _target(targets, dev, rows, width)
    given, out = out, _written(out, logits, "out")
    one = rows != 1 and isinstance(dloss, _Tensor) and dloss.dim() == 1 and dloss.shape[0] == 1
    d = _per_row(dloss, _F32, dev, 1 if one else rows, "dloss")
    _chk(lib().c6_policy_loss_grad(l, t, kind, ts, _per_row(lse, _F32, dev, rows, "lse"), _per_row(total, _F32, dev, rows, "total"), d, 0 if one else 1,
                                   out.data_ptr(), out.stride(0), _stream(dev)))
    if given is not None:
        _written_to(out)
    return out


class GradClip:
    """Global norm of gradient tensors, and the gradients scaled to at most max_norm (c6_clip):  out = g * min(1, max_norm / (norm + 1e-6)).

    Made once for buffers that stay where they are (it keeps them alive): contiguous float32 / float16 / bfloat16 tensors of one device, of any
    number and size.  outs: tensors like grads to write to; None: in place.  A graph that captured a call needs the object for as long as it is
    replayed.

    An optimizer's zero_grad() drops the gradients by default, and the next backward pass makes new ones that the object does not know: keep them with
    zero_grad(set_to_none=False)."""
    _late = []       # tables of objects that were collected: freed when the next one is made or closed, not by the collector, whose moment nobody chooses

    def __init__(self, grads, outs=None):
        grads = list(grads)
        outs = None if outs is None else list(outs)
        self.h = None
        for t in grads + (outs or []):
            if not isinstance(t, _Tensor) or not t.is_cuda or t.dtype not in _TYPE or not t.is_contiguous():
                raise C6Error("GradClip needs contiguous float32, float16 or bfloat16 tensors on the GPU")
            if t.device != grads[0].device:
                raise C6Error("GradClip's tensors live on one device")
        if not grads:
            raise C6Error("GradClip needs tensors")
        if outs is not None and (len(outs) != len(grads) or any(o.shape != g.shape or o.dtype is not g.dtype for o, g in zip(outs, grads))):
            raise C6Error("outs must be tensors like grads")
        if torch.cuda.is_current_stream_capturing():
            raise C6Error("GradClip cannot be made during a capture")
        self.device = grads[0].device
        k = len(grads)
        ptrs = (C.c_void_p * k)(*[t.data_ptr() for t in grads])
        optrs = None if outs is None else (C.c_void_p * k)(*[t.data_ptr() for t in outs])
        self._free_late()
        h = C.c_void_p()
        _chk(lib().c6_clip_create(k, ptrs, optrs, (C.c_size_t * k)(*[t.numel() for t in grads]), (C.c_int * k)(*[_TYPE[t.dtype] for t in grads]),
                                  self.device.index, C.byref(h)))
        self.h = h
        self._keep = grads, outs
        # (views of one buffer share its version)
        self._bases = list({id(b): b for b in (t if t._base is None else t._base for t in (grads if outs is None else outs))}.values())
        self._bytes = lib().c6_clip_workspace(h)

    @staticmethod
    def _free_late():
        while GradClip._late:
            try:
                h = GradClip._late.pop()
            except IndexError:      # (another thread's)
                break
            lib().c6_clip_destroy(h)      # (hipFree waits for what the device still has to do)

    def close(self):
        """frees the table once nothing that uses it runs any more"""
        if self.h:
            if torch.cuda.is_current_stream_capturing():
                raise C6Error("GradClip cannot be closed during a capture")
            self._free_late()
            h, self.h = self.h, None
            lib().c6_clip_destroy(h)
            self._keep = self._bases = None

    def __del__(self, _ending=sys.is_finalizing):
        if not _ending() and getattr(self, "h", None):
            GradClip._late.append(self.h)

    def _call(self, norm):
        if not self.h:
            raise C6Error("GradClip is closed")
        if norm is None:
            norm = torch.empty_strided((1,), (1,), dtype=_F32, device=self.device)
        elif not isinstance(norm, _Tensor) or norm.dtype is not _F32 or norm.shape != (1,) or norm.device != self.device:
            raise C6Error("norm must be a float32 tensor [1] on the gradients' device")
        else:
            _followed(norm, "norm")
        return norm, torch.empty_strided((self._bytes,), (1,), dtype=_U8, device=self.device)

    def norm(self, norm=None):
        """the global norm, a float32 tensor [1]; the gradients stay as they are"""
        given, (norm, space) = norm, self._call(norm)
        _chk(lib().c6_clip_norm(self.h, norm.data_ptr(), space.data_ptr(), self._bytes, _stream(self.device.index)))
        if given is not None:
            _written_to(norm)
        return norm

    def clip(self, max_norm, norm=None):
        """scales the gradients; returns their norm before that, a float32 tensor [1]"""
        given, (norm, space) = norm, self._call(norm)
        _chk(lib().c6_clip_apply(self.h, max_norm, norm.data_ptr(), space.data_ptr(), self._bytes, _stream(self.device.index)))
        _written_to(self._bases)
        if given is not None:
            _written_to(norm)
        return norm
