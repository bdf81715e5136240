"""dropout of a fully connected head, its mask from a counter-based generator and never stored (csrc/dropout.hip).  Part of the ``ops``
package."""
from ._lowp import *       # noqa: F401,F403  (torch, _lib and the argument helpers)

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
    if rows and cols:
        _enqueue("adv_dropout_fwd", x.device, x.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), rows, cols, _FLOATS[x.dtype],
                 p, seed, step_at, step, 1 if relu else 0)
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
    if not (rows and cols):
        return out, grad_y.new_zeros((cols,)) if with_bias else None
    gbias = ws = None
    kind = _FLOATS[grad_y.dtype]
    if with_bias:
        gbias = grad_y.new_empty((cols,))
        n = _workspace("adv_dropout_bwd_workspace_floats", rows, cols, kind)
        ws = grad_y.new_empty((n,), dtype=torch.float32) if n else None
    _enqueue("adv_dropout_bwd", grad_y.device, grad_y.data_ptr(), None if y is None else y.data_ptr(), out.data_ptr(), None if gbias is None else gbias.data_ptr(),
             None if ws is None else ws.data_ptr(), rows, cols, kind, p, seed, step_at, step)
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
        gx, gbias = dropout_bwd(grad_y.contiguous(), ctx.p, ctx.seed, ctx.step if step is None else step, y, any(ctx.needs_input_grad[4:]))      # (what follows seed may be left out)
        return gx, None, None, None, gbias, None


__all__ = [n for n in dir() if not n.startswith("__")]
