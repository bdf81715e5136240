"""matrices held in MXFP4 (32 values of a row as 4-bit floats under one power of two) and their products on the scaled matrix instructions
(csrc/mx4.hip): a fully connected head with four-bit weights, served or attacked.  Part of the ``ops`` package."""
from ._lowp import *       # noqa: F401,F403  (torch, _lib and the argument helpers)

_PANEL = 256               # columns of a panel of the layout: 128 code bytes and 8 scale bytes a row
_MOST = 1 << 20            # rows, and columns, of a matrix that the kernels index


def _fits(rows, cols, name):
    if rows > _MOST or cols > _MOST:
        raise ValueError("%s: an MXFP4 matrix has at most 2**20 rows (all leading dimensions together) and 2**20 columns, got %d x %d: take it in parts" % (name, rows, cols))


class Mx4:
    """A tensor [..., C] held in MXFP4: ``codes`` uint8 [panels, rows, 128] and ``scales`` uint8 [panels, rows, 8] (csrc/mx4.hip's layout), ``shape``
    the tensor's own.  Made by ``mx4_quantize``; ``dequantize()`` gives the values it stands for."""

    __slots__ = ("codes", "scales", "shape", "rows", "cols")

    def __init__(self, codes, scales, shape):
        shape = torch.Size(shape)
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError("an MXFP4 tensor has at least one column, got %s" % (tuple(shape),))
        self.shape, self.cols = shape, shape[-1]
        self.rows = shape.numel() // self.cols
        panels = (self.cols + _PANEL - 1) // _PANEL
        for t, name, width in ((codes, "codes", 128), (scales, "scales", 8)):
            if not (isinstance(t, torch.Tensor) and t.dtype == torch.uint8 and t.is_contiguous() and tuple(t.shape) == (panels, self.rows, width)):
                raise ValueError("%s must be a contiguous uint8 tensor [%d, %d, %d]" % (name, panels, self.rows, width))
        if codes.device != scales.device:
            raise ValueError("codes and scales are on different devices")
        self.codes, self.scales = codes, scales

    @property
    def device(self):
        return self.codes.device

    def to(self, device):
        return Mx4(self.codes.to(device), self.scales.to(device), self.shape)

    def dequantize(self, dtype=torch.float32):
        return mx4_dequantize(self, dtype)


def _made(codes, scales, shape, rows, cols):
    """an Mx4 of tensors that were laid out here: the constructor's checks are an eighth of a small quantisation's call"""
    q = Mx4.__new__(Mx4)
    q.codes, q.scales, q.shape, q.rows, q.cols = codes, scales, shape, rows, cols
    return q


def _mx4(q, name):
    if not isinstance(q, Mx4):
        raise TypeError("%s must be an Mx4 (ops.mx4_quantize)" % name)
    if not q.codes.is_cuda:
        raise TypeError("%s must be on a ROCm device (there is no CPU path)" % name)
    return q


def mx4_quantize(x):
    """``x`` [..., C] float32 / bfloat16 / float16 -> Mx4 (adv_mx4_quantize): per 32 consecutive values of a row the power of two that puts the
    largest magnitude into [4, 8), nearest 4-bit value (ties to even, beyond 6 saturated).  A block with a NaN or an infinity becomes NaN.  At most 2**20
    rows and 2**20 columns."""
    _head(x, "x")
    rows, cols = _matrix(x)
    if cols < 1:
        raise ValueError("x needs at least one column")
    _fits(rows, cols, "x")
    panels = (cols + _PANEL - 1) // _PANEL
    codes, scales = x.new_empty((panels, rows, 128), dtype=torch.uint8), x.new_empty((panels, rows, 8), dtype=torch.uint8)
    if rows:
        _enqueue("adv_mx4_quantize", x.device, x.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, cols, _FLOATS[x.dtype])
    return _made(codes, scales, x.shape, rows, cols)


def mx4_dequantize(q, dtype=torch.float32):
    """the values an Mx4 stands for, in its tensor's shape (adv_mx4_dequantize)"""
    _mx4(q, "q")
    if dtype not in _FLOATS:
        raise TypeError("dtype must be float32, bfloat16 or float16")
    x = q.codes.new_empty(q.shape, dtype=dtype)
    if q.rows:
        _enqueue("adv_mx4_dequantize", q.device, q.codes.data_ptr(), q.scales.data_ptr(), x.data_ptr(), q.rows, q.cols, _FLOATS[dtype])
    return x


def _same_device(w, *tensors):
    for t in tensors:
        if t is not None and t.device != w.device:
            raise ValueError("the operands are on different devices (%s, %s)" % (w.device, t.device))


def mx4_linear(x, w, bias=None, relu=False, dtype=None):
    """``relu?(Q(x) . W^T + bias)`` -> [..., N] (adv_mx4_linear): ``x`` [..., K] float32 / bfloat16 / float16, quantised on the way in, or an Mx4 that
    several products share (then ``dtype`` is the result's, float32 by default; else it is x's); ``w`` the Mx4 of the layer's weight [N, K];
    ``bias`` [N] of the result's type."""
    _mx4(w, "w")
    if len(w.shape) != 2:
        raise ValueError("w must be the Mx4 of a weight [N, K]")
    if isinstance(x, Mx4):
        dtype = torch.float32 if dtype is None else dtype
    else:
        _head(x, "x")
        if dtype is not None and dtype != x.dtype:
            raise TypeError("dtype is x's own unless x is an Mx4")
        dtype = x.dtype
    if dtype not in _FLOATS:
        raise TypeError("dtype must be float32, bfloat16 or float16")
    if len(x.shape) < 1 or x.shape[-1] != w.cols:
        raise ValueError("x %s does not fit a weight of %d columns" % (tuple(x.shape), w.cols))
    _same_device(w, x, bias)
    m, n, k = x.shape[:-1].numel(), w.rows, w.cols
    _fits(m, k, "x")
    y = w.codes.new_empty(x.shape[:-1] + (n,), dtype=dtype)
    if bias is not None and tuple(_head(bias, "bias", y).shape) != (n,):
        raise ValueError("bias must be [%d], got %s" % (n, tuple(bias.shape)))
    held = _mx4(x, "x") if isinstance(x, Mx4) else None
    if not (m and n):
        return y
    ws = y.new_empty((_workspace("adv_mx4_linear_workspace_bytes", m, n, k),), dtype=torch.uint8)
    _enqueue("adv_mx4_linear", y.device, x.data_ptr() if held is None else None, None if held is None else held.codes.data_ptr(),
             None if held is None else held.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), None if bias is None else bias.data_ptr(),
             y.data_ptr(), ws.data_ptr(), m, n, k, _FLOATS[dtype], 1 if relu else 0)
    return y


def mx4_linear_dgrad(grad_y, w, mask=None):
    """the gradient of ``mx4_linear`` w.r.t. ``x`` -> [..., K], straight through x's quantisation (adv_mx4_linear_dgrad): ``(0 where mask <= 0, else
    grad_y) . W`` with ``mask`` the layer's output where it had a ReLU, else None.  ``grad_y`` [..., N] float32 / bfloat16 / float16 enters exactly (bits of
    a float32 under 2**-133 are cut); sums are float32."""
    _mx4(w, "w")
    _head(grad_y, "grad_y")
    if len(w.shape) != 2 or grad_y.dim() < 1 or grad_y.shape[-1] != w.rows:
        raise ValueError("grad_y %s does not fit a weight %s" % (tuple(grad_y.shape), tuple(w.shape)))
    if mask is not None and _head(mask, "mask", grad_y).shape != grad_y.shape:
        raise ValueError("mask must have grad_y's shape")
    _same_device(w, grad_y)
    m, n, k, kind = grad_y.shape[:-1].numel(), w.rows, w.cols, _FLOATS[grad_y.dtype]
    _fits(m, k, "grad_y")
    gx = grad_y.new_empty(grad_y.shape[:-1] + (k,))
    if not m:
        return gx
    if not n:
        return gx.zero_()
    ws = gx.new_empty((_workspace("adv_mx4_linear_dgrad_workspace_bytes", m, n, k, kind),), dtype=torch.uint8)
    _enqueue("adv_mx4_linear_dgrad", gx.device, grad_y.data_ptr(), None if mask is None else mask.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
             gx.data_ptr(), ws.data_ptr(), m, n, k, kind)
    return gx


def _stamp(w):
    """moves on with every in-place change of the weight's tensors (those made in inference mode do not count theirs)"""
    return tuple(None if t.is_inference() else t._version for t in (w.codes, w.scales))


class Mx4Linear(torch.autograd.Function):
    """``Mx4Linear.apply(x, w, bias=None, relu=False)``: ``mx4_linear`` with its gradient w.r.t. ``x``; weight and bias are constants of a frozen head
    (a weight whose tensors were changed in place between the forward and the backward pass is refused, as autograd refuses it of its own)"""

    @staticmethod
    def forward(ctx, x, w, bias=None, relu=False):
        if any(ctx.needs_input_grad[2:]):            # (bias and relu may be left out)
            raise ValueError("Mx4Linear has no gradient w.r.t. its bias (a frozen head): detach it")
        y = mx4_linear(x, w, bias, relu)
        ctx.w, ctx.stamp = w, _stamp(w)
        ctx.save_for_backward(y if relu else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        y, = ctx.saved_tensors
        if _stamp(ctx.w) != ctx.stamp:
            raise RuntimeError("Mx4Linear: the weight was changed in place after the forward pass: its gradient would be another layer's")
        return mx4_linear_dgrad(grad_y.contiguous(), ctx.w, y), None, None, None


__all__ = [n for n in dir() if not n.startswith("__")]
