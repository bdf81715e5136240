"""dropout of a fully connected head, its mask from a counter-based generator and never stored (csrc/dropout.hip).  Part of the ``ops``
package."""
from ._base import *       # noqa: F401,F403  (torch, ctypes, _lib and the argument helpers)

_FLOATS = {torch.float32: _lib.ADV_F32, torch.bfloat16: _lib.ADV_BF16, torch.float16: _lib.ADV_F16}


def _head(t, name, like=None):
    """a contiguous float32 / bfloat16 / float16 ROCm tensor (of ``like``'s type and device)"""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _FLOATS and t.is_contiguous()):
        raise TypeError("%s must be a contiguous float32, bfloat16 or float16 CUDA tensor" % name)
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError("%s (%s on %s) must have the type and device of the tensor it belongs to (%s on %s)" % (name, t.dtype, t.device, like.dtype, like.device))
    return t


def _matrix(t):
    """(rows, columns) of a tensor whose last dimension is the layer's"""
    if t.dim() < 1:
        raise ValueError("a tensor of at least one dimension is needed")
    cols = t.shape[-1]
    return (t.numel() // cols if cols else 0), cols


def _draw(p, seed, step, like):
    """the generator's arguments of the C calls, checked: (p, seed, step_at, step)"""
    p, seed = float(p), int(seed)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be in [0, 1], got %r" % p)
    if not 0 <= seed < 1 << 64:
        raise ValueError("seed must be a whole number in [0, 2**64), got %d" % seed)
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != like.device:
            raise ValueError("a step tensor must hold one int64 on the tensor's device")
        return p, seed, step.data_ptr(), 0
    step = int(step)
    if not 0 <= step < 1 << 63:
        raise ValueError("step must be a whole number in [0, 2**63), got %d" % step)
    return p, seed, None, step


def dropout(x, p, seed, step=0, bias=None, relu=False, out=None):
    """``relu?(dropout(x + bias, p))`` in one pass (adv_dropout_fwd) - Linear - Dropout - ReLU of dynamic_vehicles/Model.py:24-27 behind the
    product.  ``x`` [..., C] float32 / bfloat16 / float16, ``bias`` [C] or None.  Which elements stay is a function of (``seed``, ``step``,
    the element's place) alone: give every training step and every dropout layer another ``step`` or ``seed``, and the same two to
    ``dropout_bwd``.  ``step`` may be an int64 CUDA tensor of one element, read when the kernel runs - a captured graph draws anew as it is
    moved on.  ``out`` may be ``x``."""
    _head(x, "x")
    rows, cols = _matrix(x)
    p, seed, step_at, step = _draw(p, seed, step, x)
    if bias is not None and tuple(_head(bias, "bias", x).shape) != (cols,):
        raise ValueError("bias must be [%d], got %s" % (cols, tuple(bias.shape)))
    if out is None:
        out = torch.empty_like(x)
    elif _head(out, "out", x).shape != x.shape:
        raise ValueError("out must have x's shape")
    if x.numel():
        with _on(x):
            _lib.call("adv_dropout_fwd", x.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), rows, cols, _FLOATS[x.dtype],
                      p, seed, step_at, step, 1 if relu else 0, _stream(x))
    return out


def dropout_bwd(grad_y, p, seed, step=0, y=None, with_bias=False, out=None):
    """(gradient w.r.t. ``x``, gradient w.r.t. ``bias`` or None) of ``dropout`` called with the same ``p``, ``seed`` and ``step`` (adv_dropout_bwd).
    ``y``: the forward's result, needed if and only if it had ``relu``.  The bias gradient is summed in float32 in a fixed order.  ``out`` may
    be ``grad_y``."""
    _head(grad_y, "grad_y")
    rows, cols = _matrix(grad_y)
    p, seed, step_at, step = _draw(p, seed, step, grad_y)
    if y is not None and _head(y, "y", grad_y).shape != grad_y.shape:
        raise ValueError("y must have grad_y's shape")
    if out is None:
        out = torch.empty_like(grad_y)
    elif _head(out, "out", grad_y).shape != grad_y.shape:
        raise ValueError("out must have grad_y's shape")
    if not grad_y.numel():
        return out, torch.zeros((cols,), dtype=grad_y.dtype, device=grad_y.device) if with_bias else None
    gbias = ws = None
    with _on(grad_y):
        if with_bias:
            gbias = torch.empty((cols,), dtype=grad_y.dtype, device=grad_y.device)
            n = _lib.load().adv_dropout_bwd_workspace_floats(rows, cols, _FLOATS[grad_y.dtype])
            ws = torch.empty((n,), dtype=torch.float32, device=grad_y.device) if n > 0 else None
        _lib.call("adv_dropout_bwd", grad_y.data_ptr(), None if y is None else y.data_ptr(), out.data_ptr(), None if gbias is None else gbias.data_ptr(),
                  None if ws is None else ws.data_ptr(), rows, cols, _FLOATS[grad_y.dtype], p, seed, step_at, step, _stream(grad_y))
    return out, gbias


class Dropout(torch.autograd.Function):
    """``Dropout.apply(x, p, seed, step=0, bias=None, relu=False)``: ``dropout`` with its gradients w.r.t. ``x`` and ``bias``.  A ``step`` tensor must
    not be changed between the forward and the backward pass (autograd refuses the backward then)."""

    @staticmethod
    def forward(ctx, x, p, seed, step=0, bias=None, relu=False):
        y = dropout(x, p, seed, step, bias, relu)
        tensor_step = isinstance(step, torch.Tensor)
        ctx.save_for_backward(y if relu else None, step if tensor_step else None)
        ctx.p, ctx.seed, ctx.step = p, seed, None if tensor_step else step
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        y, step = ctx.saved_tensors
        gx, gbias = dropout_bwd(grad_y.contiguous(), ctx.p, ctx.seed, ctx.step if step is None else step, y, ctx.needs_input_grad[4])
        return gx, None, None, None, gbias, None


__all__ = [n for n in dir() if not n.startswith("__")]
