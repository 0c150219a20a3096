"""Operators of a net in front of a conditional flow (``nessai_amd.ops``).

The reference hands a conditional flow any ``context`` tensor (``src/nessai/flows/base.py:236-245``) and leaves the net
that makes it to torch.  What such a net is built from and trained with has kernels here:

=======================  ===================================================================================
``embedding``            rows of a table by label, scaled; the gradient by sorted tokens
``group_norm_act``       group norm over the last (channel) dimension with an activation, and its backward pass
``grad_norm``            the norm over many gradient tensors
``clip_grad_norm_``      the same, then the clip (``torch.nn.utils.clip_grad_norm_`` of the reference's training
                         loop, ``src/nessai/flowmodel/base.py:437-441``)
=======================  ===================================================================================

Values are float32, bfloat16 or float16; sums and statistics are held in float32 or wider and results are rounded once.
There is no CPU implementation; float64 is refused, never cast down.  Derivatives are first-order and reverse-mode: a tensor
with a tangent (``torch.autograd.forward_ad``, ``torch.func.jvp``) is refused.  Every call enqueues on the current stream of the
tensors' device, waits for nothing (but ``error_if_nonfinite``) and may be captured into a HIP graph.  The functions here name
the arguments; ``csrc/nsa_torch.cpp`` checks them, allocates and records for autograd.  Meta and fake tensors give the results'
shapes, so that the operators can be traced (``torch.compile``; the first call loads the library and is made outside).
"""

import math

import torch

from . import lib

_NORMS = {1.0: 1, 2.0: 2, math.inf: 3}  # NSA_NORM_* (include/nessai_amd.h)
_ACTIVATIONS = {None: -1, "relu": 0, "tanh": 1, "silu": 2, "swish": 2}  # NSA_FN_*


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """Group norm over the channels of a channels-last tensor, followed by an activation.

    ``x``: ``(N, ..., C)``; the mean and the (biased) variance are taken for every sample and each of the
    ``num_groups`` groups of ``C / num_groups`` neighbouring channels, over all positions between the first and the
    last dimension.  ``weight`` / ``bias``: ``(C,)``, float32 or of ``x``'s type, or ``None``.  ``activation``:
    ``None``, ``"relu"``, ``"tanh"`` or ``"silu"``, as the flows' conditioners have them.  Differentiable once in ``x``,
    ``weight`` and ``bias``.  A tensor that is not contiguous is copied first; the result is contiguous.  At most ``2**30``
    channels.
    """
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Unknown activation: {activation}")
    lib.load_torch()
    return torch.ops.nessai_amd.group_norm_act(x, num_groups, weight, bias, eps, _ACTIVATIONS[activation])


def embedding(indices, weight, scale=1.0, padding_idx=None):
    """``weight[indices] * scale``: rows of a ``(V, D)`` table, ``indices`` int32 or int64 of any shape.

    The gradient of ``weight`` is dense; its rows are float32 sums over the tokens in a fixed order (equal inputs give equal
    bits), rounded once.  Row ``padding_idx`` gets none.  An index outside ``[0, V)`` cannot be seen without waiting for
    the device: its row of the result is NaN, and it takes no part in the gradient.  Differentiable once.  At most
    ``2**31 - 1`` rows and indices and ``2**20`` columns.
    """
    lib.load_torch()
    return torch.ops.nessai_amd.embedding(indices, weight, scale, padding_idx)


def _norm_code(norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or inf (got {norm_type})")
    return code


def grad_norm(tensors, norm_type=2.0):
    """The norm of all elements of ``tensors`` together (``torch.nn.utils.get_total_norm``): a float32 scalar on their
    device.  ``norm_type``: 1, 2 or ``inf``.  A tensor that is listed twice counts twice."""
    lib.load_torch()
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    return torch.ops.nessai_amd.grad_norm(tensors, _norm_code(norm_type))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scale the gradients of ``parameters`` in place so that their norm over all of them is at most ``max_norm``; returns
    the norm before, a float32 scalar on their device.

    As ``torch.nn.utils.clip_grad_norm_``: the factor is ``min(1, max_norm / (norm + 1e-6))``, parameters without a
    gradient are passed over, and a norm that is not finite scales like any other unless ``error_if_nonfinite`` (which
    waits for the device).  ``norm_type``: 1, 2 or ``inf``.  Gradients may be of several types, but not overlap in memory.
    """
    lib.load_torch()
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    args = (_norm_code(norm_type), max_norm, error_if_nonfinite)
    if torch.compiler.is_compiling():  # (the gradients as arguments: the compiled graph must show what changes)
        return torch.ops.nessai_amd.clip_grad_norm_of_([p.grad for p in parameters if p.grad is not None], *args)
    return torch.ops.nessai_amd.clip_grad_norm_(parameters, *args)
