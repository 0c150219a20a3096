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
There is no CPU implementation; float64 is refused, never cast down.  Every call enqueues on the current stream of the
tensors' device, waits for nothing and may be captured into a HIP graph.
"""

import math

import torch
from torch.autograd.function import once_differentiable

from . import lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # NSA_DT_* (include/nessai_amd.h)
_NORMS = {1.0: 1, 2.0: 2, math.inf: 3}  # NSA_NORM_*
_ACTIVATIONS = {None: -1, "relu": 0, "tanh": 1, "silu": 2, "swish": 2}  # NSA_FN_*


def _dtype_code(t, what):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16 (got {t.dtype}): there is no kernel for other "
                        "types, and nothing is cast down silently")
    return code


def _on_device(t, what):
    if t.device.type != "cuda":
        raise RuntimeError(f"{what}: nessai_amd operators take tensors on a ROCm device (got {t.device}); there is no CPU "
                           "fallback")


def _call(device, name, *args):
    """The C entry point ``name`` on the current stream of ``device``."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(device, name, *args)
    stream = torch.cuda.current_stream(device).cuda_stream
    lib.check(getattr(lib.load(), name)(*args, stream), name)


def _workspace(device, size):
    return torch.empty(size, dtype=torch.uint8, device=device)


# -- group norm with an activation ----------------------------------------------------------


def _rows(x):
    """``(samples, positions)`` of a channels-last tensor."""
    return x.shape[0], math.prod(x.shape[1:-1])


def _group_norm_forward(x, groups, weight, bias, eps, activation):
    samples, length = _rows(x)
    channels, code = x.shape[-1], _DTYPES[x.dtype]
    y = torch.empty_like(x)
    stats = torch.empty((2, samples, groups), dtype=torch.float32, device=x.device)
    if x.numel():
        kind = weight if weight is not None else bias
        size = lib.load().nsa_group_norm_workspace(samples, length, channels, groups, code, 0)
        ws = _workspace(x.device, size)
        mean = stats.data_ptr()
        _call(x.device, "nsa_group_norm_forward", samples, length, channels, groups, code, x.data_ptr(),
              0 if kind is None else _DTYPES[kind.dtype], None if weight is None else weight.data_ptr(),
              None if bias is None else bias.data_ptr(), eps, activation, y.data_ptr(), mean,
              mean + 4 * samples * groups, ws.data_ptr(), size)
    return y, stats


def _group_norm_backward(x, dy, groups, weight, bias, activation, stats, want_dx, want_dw, want_db):
    samples, length = _rows(x)
    channels, code = x.shape[-1], _DTYPES[x.dtype]
    kind = weight if weight is not None else bias
    dx = torch.empty_like(x) if want_dx else None
    dw = torch.empty_like(weight) if want_dw else None
    db = torch.empty_like(bias) if want_db else None
    size = lib.load().nsa_group_norm_workspace(samples, length, channels, groups, code, 1)
    ws = _workspace(x.device, size)
    mean = stats.data_ptr()
    _call(x.device, "nsa_group_norm_backward", samples, length, channels, groups, code, x.data_ptr(), dy.data_ptr(),
          0 if kind is None else _DTYPES[kind.dtype], None if weight is None else weight.data_ptr(),
          None if bias is None else bias.data_ptr(), activation, mean, mean + 4 * samples * groups,
          None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
          None if db is None else db.data_ptr(), ws.data_ptr(), size)
    return dx, dw, db


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation):
        y, stats = _group_norm_forward(x, groups, weight, bias, eps, activation)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.activation = groups, activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = _group_norm_backward(x, dy.contiguous(), ctx.groups, weight, bias, ctx.activation, stats, *need[:3])
        return (*grads, None, None, None)


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """Group norm over the channels of a channels-last tensor, followed by an activation.

    ``x``: ``(N, ..., C)``; the mean and the (biased) variance are taken for every sample and each of the
    ``num_groups`` groups of ``C / num_groups`` neighbouring channels, over all positions between the first and the
    last dimension.  ``weight`` / ``bias``: ``(C,)``, float32 or of ``x``'s type, or ``None``.  ``activation``:
    ``None``, ``"relu"``, ``"tanh"`` or ``"silu"``, as the flows' conditioners have them.  Differentiable once in ``x``,
    ``weight`` and ``bias``.  A tensor that is not contiguous is copied first; the result is contiguous.
    """
    if x.dim() < 2:
        raise ValueError(f"expected a tensor of shape (N, ..., C), got {tuple(x.shape)}")
    _dtype_code(x, "group_norm_act: x")
    groups, channels = int(num_groups), x.shape[-1]
    if groups < 1 or channels < 1 or channels % groups:
        raise ValueError(f"{channels} channels cannot be divided into {num_groups} groups")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Unknown activation: {activation}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative (got {eps})")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (channels,):
            raise ValueError(f"expected a {name} of shape ({channels},), got {tuple(p.shape)}")
        if p.dtype != torch.float32 and p.dtype != x.dtype:
            raise TypeError(f"group_norm_act: {name} must be float32 or of x's type {x.dtype} (got {p.dtype})")
        if p.device != x.device:
            raise ValueError(f"group_norm_act: {name} is on {p.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("group_norm_act: weight and bias must have one type")
    _on_device(x, "group_norm_act")
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    code = _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _GroupNormAct.apply(x, weight, bias, groups, eps, code)
    return _group_norm_forward(x, groups, weight, bias, eps, code)[0]


# -- embedding ------------------------------------------------------------------------------


def _embedding_forward(ids, weight, scale):
    vocab, width = weight.shape
    out = torch.empty((*ids.shape, width), dtype=weight.dtype, device=weight.device)
    if out.numel():
        _call(weight.device, "nsa_embedding_forward", ids.numel(), vocab, width, _DTYPES[weight.dtype], ids.data_ptr(),
              ids.element_size(), weight.data_ptr(), scale, out.data_ptr())
    return out


def _embedding_backward(ids, dy, shape, scale, padding):
    vocab, width = shape
    code = _DTYPES[dy.dtype]
    dweight = torch.empty(shape, dtype=dy.dtype, device=dy.device)
    size = lib.load().nsa_embedding_workspace(ids.numel(), vocab, width, code)
    ws = _workspace(dy.device, size)
    _call(dy.device, "nsa_embedding_backward", ids.numel(), vocab, width, code, ids.data_ptr(), ids.element_size(),
          dy.data_ptr(), scale, padding, dweight.data_ptr(), ws.data_ptr(), size)
    return dweight


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding):
        ctx.save_for_backward(ids)
        ctx.shape, ctx.scale, ctx.padding = weight.shape, scale, padding
        return _embedding_forward(ids, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        return _embedding_backward(ids, dy.contiguous(), ctx.shape, ctx.scale, ctx.padding), None, None, None


def embedding(indices, weight, scale=1.0, padding_idx=None):
    """``weight[indices] * scale``: rows of a ``(V, D)`` table, ``indices`` int32 or int64 of any shape.

    The gradient of ``weight`` is dense; its rows are float32 sums over the tokens in their order (equal inputs give equal
    bits), rounded once.  Row ``padding_idx`` gets none.  An index outside ``[0, V)`` cannot be seen without waiting for
    the device: its row of the result is NaN, and it takes no part in the gradient.
    """
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"embedding: indices must be int32 or int64 (got {indices.dtype})")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"embedding: expected a table of shape (V, D), got {tuple(weight.shape)}")
    _dtype_code(weight, "embedding: weight")
    vocab = weight.shape[0]
    if vocab >= 2**31 or indices.numel() >= 2**31:
        raise ValueError("embedding: at most 2**31 - 1 rows and indices")
    padding = -1
    if padding_idx is not None:
        padding = int(padding_idx)
        if not -vocab <= padding < vocab:
            raise ValueError(f"embedding: padding_idx {padding_idx} is outside a table of {vocab} rows")
        padding %= vocab
    if indices.device != weight.device:
        raise ValueError(f"embedding: indices are on {indices.device}, weight on {weight.device}")
    _on_device(weight, "embedding")
    ids, scale = indices.contiguous(), float(scale)
    weight = weight.contiguous()
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(weight, ids, scale, padding)
    return _embedding_forward(ids, weight, scale)


# -- the norm over many gradients, and the clip ---------------------------------------------


def _dense(t):
    """Whether the elements of ``t`` fill one stretch of memory without gaps or repeats, in whatever order."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _norm_code(norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or inf (got {norm_type})")
    return code


def _checked(tensors, what):
    for t in tensors:
        if t.layout != torch.strided:
            raise TypeError(f"{what}: gradients must be dense (got {t.layout})")
        _dtype_code(t, f"{what}: gradients")
    devices = {t.device for t in tensors}
    if len(devices) > 1:
        raise ValueError(f"{what}: gradients on several devices: {sorted(map(str, devices))}")
    _on_device(tensors[0], what)
    return tensors[0].device


def _norm_call(name, tensors, kind, *factor):
    device, count = tensors[0].device, len(tensors)
    L = lib.load()
    out = torch.empty((), dtype=torch.float32, device=device)
    size = L.nsa_grad_norm_workspace(count)
    ws = _workspace(device, size)
    ptrs = (lib.c_void_p * count)(*[t.data_ptr() for t in tensors])
    sizes = (lib.c_ll * count)(*[t.numel() for t in tensors])
    codes = (lib.c_int * count)(*[_DTYPES[t.dtype] for t in tensors])
    _call(device, name, count, ptrs, sizes, codes, kind, *factor, ws.data_ptr(), size, out.data_ptr())
    return out


def grad_norm(tensors, norm_type=2.0):
    """The norm of all elements of ``tensors`` together (``torch.nn.utils.get_total_norm``): a float32 scalar on their
    device.  ``norm_type``: 1, 2 or ``inf``.  A tensor that is listed twice counts twice."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    kind = _norm_code(norm_type)
    if not tensors:
        return torch.tensor(0.0)
    _checked(tensors, "grad_norm")
    with torch.no_grad():
        return _norm_call("nsa_grad_norm", [t if _dense(t) else t.contiguous() for t in tensors], kind)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Scale the gradients of ``parameters`` in place so that their norm over all of them is at most ``max_norm``; returns
    the norm before, a float32 scalar on their device.

    As ``torch.nn.utils.clip_grad_norm_``: the factor is ``min(1, max_norm / (norm + 1e-6))``, parameters without a
    gradient are passed over, and a norm that is not finite scales like any other unless ``error_if_nonfinite`` (which
    waits for the device).  ``norm_type``: 1, 2 or ``inf``.  Gradients may be of several types, but not overlap in memory.
    """
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    kind, max_norm = _norm_code(norm_type), float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN (got {max_norm})")
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    _checked(grads, "clip_grad_norm_")
    # a gradient with gaps between its elements is clipped in a copy; one whose elements share memory cannot be
    gaps = [g for g in grads if not _dense(g)]
    for g in gaps:
        if any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
            raise ValueError("clip_grad_norm_: a gradient's elements overlap in memory (an expanded tensor); clone it")
    with torch.no_grad():
        copies = [g.contiguous() for g in gaps]
        dense = [g for g in grads if _dense(g)] + copies if gaps else grads
        if error_if_nonfinite:
            norm = _norm_call("nsa_grad_norm", dense, kind)
            if not math.isfinite(float(norm)):
                raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so "
                                   "it cannot be clipped")
        norm = _norm_call("nsa_grad_clip", dense, kind, max_norm)
        for g, c in zip(gaps, copies):
            g.copy_(c)
        # the kernels wrote behind torch's back: graphs that saved a gradient must see that it changed
        torch.autograd.graph.increment_version(grads)
    return norm
