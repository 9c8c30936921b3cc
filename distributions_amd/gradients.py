"""The list of gradients that sum_logpdf_grad and its relatives return: its 2-norm over all tensors, and clipping by it.

Gradients are torch CUDA tensors of one device (float64, float32, float16, bfloat16, mixed as they come, any strides) or
NumPy arrays; None entries (arguments that are data) are passed over.  Squares are added in float64 in a fixed order.  The
norm is float32 if every gradient is at most 32 bits wide, else float64.  csrc/m355_gradnorm.hip."""

from ._gradnorm import clip_global_norm as _clip
from ._gradnorm import global_norm as _norm


def global_norm(grads):
    """sqrt(sum of the squares of all elements of all gradients): a 0-d tensor on the device (NumPy inputs: a float).  A
    tensor that is listed twice counts twice; an empty list has norm 0."""
    return _norm(grads)


def clip_global_norm(grads, max_norm, out=None):
    """(norm, clipped gradients): every gradient times max_norm / norm where norm > max_norm, unchanged otherwise and where
    the norm that is returned is not finite (nothing is scaled by 0 or NaN: the caller sees the norm; a float32 norm is
    infinite from 3.4e38 on).  max_norm is a number >= 0.  out: list
    of tensors that receive the result, in the gradients' order; out=grads clips in place.  Outputs that share memory with
    each other or with another gradient are refused."""
    return _clip(grads, max_norm, out)
