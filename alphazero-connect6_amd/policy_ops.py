"""Operators on a policy's logits and on gradients, for device tensors (include/connect6_amd.h part 7): what logits go through before a
move is chosen, the loss they are trained on, and the clipping of the gradients it sends back.

    y = logits_process(logits, mask=mask, bias=bias, history=moves, history_len=lens, penalties=p)
    loss, lse, total, grad = policy_loss(logits, targets, mask=mask, grad_scale=1.0 / rows)
    norm = GradClip(grads).clip(1.0)

Everything runs on torch's current stream of the tensors' device without synchronising, and can be captured into a graph.  Arguments
that do not fit raise C6Error before anything runs.  Nothing here is recorded by autograd: logits that require a gradient are refused
(pass them detached; policy_loss returns the gradient, policy_loss_grad takes the upstream one).

`import torch` comes before the first use of the library in a process that wants both on the GPU: whichever is first brings the HIP runtime
that the other then shares (torch does not start on another's)."""
import ctypes as C

import torch

import alphazero_connect6_amd as _pkg

from . import C6Error, Logits, _chk, lib

if _pkg._lib is not None and _pkg.device_count() > 0 and not torch.cuda.is_available():
    raise C6Error("libconnect6_amd was used before torch was imported: torch cannot share its HIP runtime; import torch first")

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INDEX = {torch.int32: 0, torch.int64: 1}
_WEIGHTS = 2


def _need(ok, message):
    if not ok:
        raise C6Error(message)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _logits(x, mask):
    """-> (c6_logits, rows, width)"""
    _need(isinstance(x, torch.Tensor) and x.is_cuda and x.dim() == 2 and x.dtype in _TYPE,
          "logits must be a [rows, width] tensor of float32, float16 or bfloat16 on the GPU")
    rows, width = x.shape
    stride, step = x.stride()
    _need(step == 1 or width <= 1, "the entries of a row of logits must lie next to each other")
    _need(not x.requires_grad, "logits that require a gradient: autograd does not see this operator, pass logits.detach()")
    device = x.get_device()
    if mask is None:
        return Logits(rows, width, _TYPE[x.dtype], device, x.data_ptr(), stride, None, 0, 0), rows, width
    _need(isinstance(mask, torch.Tensor) and mask.dtype is torch.uint8 and mask.get_device() == device, "mask must be a uint8 tensor on the logits' device")
    if mask.dim() == 1:
        mask = mask.unsqueeze(0)
    nb = (width + 7) // 8
    _need(mask.dim() == 2 and mask.shape[1] == nb and mask.shape[0] in (rows, 1),
          f"mask must be [{rows}, {nb}] (or [1, {nb}], [{nb}]): one bit per entry of logits, entry v at bit v % 8 of byte v // 8")
    row, byte = mask.stride()
    return Logits(rows, width, _TYPE[x.dtype], device, x.data_ptr(), stride, mask.data_ptr(), 0 if mask.shape[0] == 1 else row, byte), rows, width


def _written(out, x, rows, width, what):
    if out is None:
        return torch.empty((rows, width), dtype=x.dtype, device=x.device)
    _need(isinstance(out, torch.Tensor) and out.get_device() == x.get_device() and out.dtype is x.dtype and out.shape == x.shape,
          f"{what} must have the logits' shape, type and device")
    _need(out.stride(1) == 1 or width <= 1, f"the entries of a row of {what} must lie next to each other")
    return out


def _rows_by(t, dtype, device, rows, width, what):
    """(pointer, row stride) of a [rows, width] / [1, width] / [width] tensor"""
    _need(isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == device, f"{what} must be a {dtype} tensor on the logits' device")
    if t.dim() == 1:
        t = t.unsqueeze(0)
    _need(t.dim() == 2 and t.shape[1] == width and t.shape[0] in (rows, 1), f"{what} must be [{rows}, {width}], [1, {width}] or [{width}]")
    _need(t.stride(1) == 1 or width <= 1, f"the entries of a row of {what} must lie next to each other")
    return t.data_ptr(), 0 if t.shape[0] == 1 else t.stride(0)


def _per_row(t, device, rows, what):
    _need(isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.get_device() == device and t.shape == (rows,) and (rows <= 1 or t.stride(0) == 1),
          f"{what} must be a contiguous float32 tensor [{rows}] on the logits' device")
    return t.data_ptr()


def logits_process(logits, mask=None, bias=None, history=None, history_len=None, penalties=None, out=None):
    """Penalties for repeated moves (or tokens), a bias and a mask on logits [rows, width] (c6_logits_process):

        y = x;  if v occurs c > 0 times in the row's history:  y = (x > 0 ? x / repetition : x * repetition) - (frequency * c + presence)
        y += bias;  an entry that is not legal becomes -infinity

    mask: uint8 [rows, ceil(width / 8)], any strides (a transposed view of legal_mask's layout too), or one for all rows; set bits are legal.
    bias: float32 [width] or [rows, width].  history: int32 [rows, cap] ids (or one for all rows), of which the first history_len[r] count (int32
    [rows]; None: all); ids outside the row, such as -1, count for nothing.  penalties: float32 [3] or [rows, 3] = repetition, frequency, presence.
    out: a tensor like logits, possibly logits itself.  Returns out."""
    l, rows, width = _logits(logits, mask)
    dev = l.device
    out = _written(out, logits, rows, width, "out")
    h = n = p = b = None
    hs = ps = bs = cap = 0
    if history is not None:
        _need(isinstance(history, torch.Tensor) and history.dim() in (1, 2), "history must be an int32 tensor [rows, cap] or [cap]")
        cap = history.shape[-1]
        h, hs = _rows_by(history, torch.int32, dev, rows, cap, "history")
        _need(penalties is not None, "a history needs penalties")
        p, ps = _rows_by(penalties, torch.float32, dev, rows, 3, "penalties")
        if history_len is not None:
            _need(isinstance(history_len, torch.Tensor) and history_len.dtype is torch.int32 and history_len.get_device() == dev
                  and history_len.shape == (rows,) and (rows <= 1 or history_len.stride(0) == 1), f"history_len must be a contiguous int32 tensor [{rows}]")
            n = history_len.data_ptr()
    else:
        _need(history_len is None and penalties is None, "history_len and penalties need a history")
    if bias is not None:
        b, bs = _rows_by(bias, torch.float32, dev, rows, width, "bias")
    _chk(lib().c6_logits_process(l, h, hs, n, cap, p, ps, b, bs, out.data_ptr(), out.stride(0), _stream(dev)))
    return out


def _target(targets, device, rows, width):
    """-> (pointer, kind, stride)"""
    _need(isinstance(targets, torch.Tensor) and targets.get_device() == device, "targets must be a tensor on the logits' device")
    if targets.dtype in _INDEX:
        _need(targets.shape == (rows,) and (rows <= 1 or targets.stride(0) == 1), f"targets of indices must be contiguous, [{rows}]")
        return targets.data_ptr(), _INDEX[targets.dtype], 0
    _need(targets.dtype is torch.float32 and targets.dim() == 2 and targets.shape == (rows, width),
          f"targets must be int32 or int64 indices [{rows}], or float32 weights [{rows}, {width}]")
    _need(targets.stride(1) == 1 or width <= 1, "the weights of a row must lie next to each other")
    return targets.data_ptr(), _WEIGHTS, targets.stride(0)


def policy_loss(logits, targets, mask=None, grad_scale=None, grad=None):
    """Cross entropy of logits [rows, width] against targets over the legal entries (c6_policy_loss) -> (loss, lse, total), float32 [rows] each, or
    (loss, lse, total, gradient) with a grad_scale (the derivative of grad_scale * sum(loss) by the logits, in the logits' type; 1 / rows for a mean).

    targets: int32 / int64 [rows] -- the entry played; outside the row or illegal: the row adds nothing -- or float32 [rows, width] weights >= 0
    (visit counts, a teacher's distribution).  loss = sum t (lse - x), total = sum t.  mask as in logits_process.  grad: where the gradient goes,
    possibly logits itself.  A row with no legal entry above -infinity has loss 0, lse -infinity and gradient 0."""
    l, rows, width = _logits(logits, mask)
    dev = l.device
    t, kind, ts = _target(targets, dev, rows, width)
    stats = torch.empty((3, rows), dtype=torch.float32, device=logits.device)
    g, gs = None, 0
    if grad_scale is not None:
        grad = _written(grad, logits, rows, width, "grad")
        g, gs = grad.data_ptr(), grad.stride(0)
    else:
        _need(grad is None, "grad needs a grad_scale")
        grad_scale = 0.0
    L = lib()
    nbytes = L.c6_policy_loss_workspace(rows, width)
    space = torch.empty(nbytes, dtype=torch.uint8, device=logits.device) if nbytes else None
    at = stats.data_ptr()
    _chk(L.c6_policy_loss(l, t, kind, ts, at, at + 4 * rows, at + 8 * rows, g, gs, grad_scale, space.data_ptr() if nbytes else None, nbytes, _stream(dev)))
    loss, lse, total = stats.unbind(0)
    return (loss, lse, total) if g is None else (loss, lse, total, grad)


def policy_loss_grad(logits, targets, lse, total, dloss, mask=None, out=None):
    """The gradient by the logits from the lse and total of policy_loss and the upstream gradient dloss, float32 [rows] or [1] (c6_policy_loss_grad).
    out: where it goes, possibly logits itself."""
    l, rows, width = _logits(logits, mask)
    dev = l.device
    t, kind, ts = _target(targets, dev, rows, width)
    out = _written(out, logits, rows, width, "out")
    one = isinstance(dloss, torch.Tensor) and dloss.shape == (1,) and rows != 1
    d = _per_row(dloss, dev, 1 if one else rows, "dloss")
    _chk(lib().c6_policy_loss_grad(l, t, kind, ts, _per_row(lse, dev, rows, "lse"), _per_row(total, dev, rows, "total"), d, 0 if one else 1, out.data_ptr(),
                                   out.stride(0), _stream(dev)))
    return out


class GradClip:
    """Global norm of gradient tensors, and the gradients scaled to at most max_norm (c6_clip):  out = g * min(1, max_norm / (norm + 1e-6)).

    Made once for buffers that stay where they are (it keeps them alive): contiguous float32 / float16 / bfloat16 tensors of one device, of any
    number and size.  outs: tensors like grads to write to; None: in place.  A graph that captured a call needs the object for as long as it is
    replayed."""
    _late = []       # tables of objects that were collected during a capture, where memory cannot be freed

    def __init__(self, grads, outs=None):
        grads = list(grads)
        outs = None if outs is None else list(outs)
        self.h = None
        _need(grads and all(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _TYPE and t.is_contiguous() for t in grads + (outs or [])),
              "GradClip needs contiguous float32, float16 or bfloat16 tensors on the GPU")
        self.device = grads[0].device
        _need(all(t.device == self.device for t in grads + (outs or [])), "GradClip's tensors live on one device")
        if outs is not None:
            _need(len(outs) == len(grads) and all(o.shape == g.shape and o.dtype is g.dtype for o, g in zip(outs, grads)), "outs must be tensors like grads")
        k = len(grads)
        ptrs = (C.c_void_p * k)(*[t.data_ptr() for t in grads])
        optrs = None if outs is None else (C.c_void_p * k)(*[t.data_ptr() for t in outs])
        h = C.c_void_p()
        _chk(lib().c6_clip_create(k, ptrs, optrs, (C.c_size_t * k)(*[t.numel() for t in grads]), (C.c_int * k)(*[_TYPE[t.dtype] for t in grads]),
                                  self.device.index, C.byref(h)))
        self.h = h
        self._keep = grads, outs
        self._bytes = lib().c6_clip_workspace(h)

    def close(self):
        """frees the table once nothing that uses it runs any more"""
        if getattr(self, "h", None):
            _need(not torch.cuda.is_current_stream_capturing(), "GradClip cannot be closed during a capture")
            torch.cuda.synchronize(self.device)
            while GradClip._late:
                lib().c6_clip_destroy(GradClip._late.pop())
            lib().c6_clip_destroy(self.h)
            self.h = self._keep = None

    def __del__(self):
        if getattr(self, "h", None) and torch.cuda.is_current_stream_capturing():
            GradClip._late.append(self.h)
        else:
            self.close()

    def _call(self, norm):
        _need(self.h is not None, "GradClip is closed")
        if norm is None:
            norm = torch.empty(1, dtype=torch.float32, device=self.device)
        _need(isinstance(norm, torch.Tensor) and norm.dtype is torch.float32 and norm.shape == (1,) and norm.device == self.device,
              "norm must be a float32 tensor [1] on the gradients' device")
        return norm, torch.empty(self._bytes, dtype=torch.uint8, device=self.device)

    def norm(self, norm=None):
        """the global norm, a float32 tensor [1]; the gradients stay as they are"""
        norm, space = self._call(norm)
        _chk(lib().c6_clip_norm(self.h, norm.data_ptr(), space.data_ptr(), self._bytes, _stream(self.device)))
        return norm

    def clip(self, max_norm, norm=None):
        """scales the gradients; returns their norm before that, a float32 tensor [1]"""
        norm, space = self._call(norm)
        _chk(lib().c6_clip_apply(self.h, max_norm, norm.data_ptr(), space.data_ptr(), self._bytes, _stream(self.device)))
        return norm
