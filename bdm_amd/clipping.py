"""The global norm of a model's gradients, and their clipping.

The shell's optimizer clips with ``torch.nn.utils.clip_grad_norm_``
(reproduction/experiments/optim.py:33-36), whose norm of BF16 gradients is
itself a BF16 number: up to 2^-9 of it off, and the clipped gradients with it.
Here one pass over all tensors forms the norm from FP64 sums, and one more
scales them.
"""

from __future__ import annotations

from torch import Tensor

from . import ops


def gradient_norm(gradients) -> Tensor:
    """sqrt of the sum of squares over all tensors, an FP32 scalar.

    gradients: BF16 or FP32 tensors on one ROCm device, any shapes and any mix
    of the two; None is passed over (a parameter without a gradient), and a
    tensor that is there twice counts twice.  Without tensors the norm is 0 (on
    the CPU).  The sums are FP64 and made in a fixed order: they neither overflow
    nor vanish, and repeat bit for bit."""
    return ops.gradient_norm(gradients)


def clip_gradients(gradients, max_norm: float, *, out=None) -> Tensor:
    """Scales the gradients by min(1, max_norm / (norm + 1e-6)) and returns their
    norm before that, ``gradient_norm(gradients)``.

    In place by default; ``out`` gives a tensor for each gradient instead, of as
    many elements in the same order, BF16 or FP32 (an optimizer's FP32 gradients, for instance).  Each value
    is rounded once.  A norm of infinity gives the factor 0 and one of NaN the
    factor NaN, as torch's clipping does without its check.  To autograd it is an
    in-place operation on the tensors written.  A tensor written may
    not share memory with another one of the call (ValueError), so that none is
    given twice.  The host is not synchronised."""
    return ops.clip_gradients(gradients, max_norm, out=out)
