"""what ``dropout`` and ``mx4`` share: the three types of a fully connected head, the checks of its tensors, and a short way to the library (these
calls take a few microseconds on the device: half a dozen small Python calls in front of each would be the larger part)."""
import functools

from ._base import *       # noqa: F401,F403  (torch, _lib)

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


def _enqueue(name, device, *args):
    """``name``(*args, the device's current stream) with ``device`` current"""
    lib, index = _lib.load(), device.index
    if torch.cuda.current_device() == index:
        code = getattr(lib, name)(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = getattr(lib, name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _lib.check(name, code)


@functools.lru_cache(maxsize=4096)
def _workspace(query, *sizes):
    """what a ``*_workspace_*`` query says for these sizes (a function of the sizes alone)"""
    n = getattr(_lib.load(), query)(*sizes)
    if n < 0:
        _lib.check(query, n)
    return n


__all__ = [n for n in dir() if not n.startswith("__")]
