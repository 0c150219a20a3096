"""A conditional flow with a trainable net in front of its context.

The reference's conditional flows take the ``context`` as it is (``src/nessai/flows/base.py:236-245``); nflows' ``Flow``,
which they are built on, also takes an ``embedding_net`` that makes the context from what the user has.  ``ContextFlow`` is
that flow here, and ``ContextNet`` a net for what conditional inputs usually are: labels (which detector, which model class,
which event) and continuous columns.  The net's parts are the operators of ``nessai_amd.ops``; its linear layers are plain
matrix products.
"""

import math

import torch
from torch import nn

from .. import ops
from .base import DIR_FORWARD, MODE_APPLY, MODE_LOGPROB, BaseFlow, HipFlow
from .modules import activation_name


class Embedding(nn.Module):
    """Rows of a ``(num_embeddings, features)`` table times ``sqrt(features)`` (``ops.embedding``): the table's entries start
    at the scale of a linear layer's weights, the rows at that of its outputs."""

    def __init__(self, num_embeddings, features, padding_idx=None):
        super().__init__()
        self.padding_idx = padding_idx
        self.scale = math.sqrt(features)
        self.weight = nn.Parameter(torch.empty(num_embeddings, features))
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.normal_(self.weight, std=1.0 / self.scale)
        if self.padding_idx is not None:
            with torch.no_grad():
                self.weight[self.padding_idx].zero_()

    def forward(self, indices):
        return ops.embedding(indices, self.weight, scale=self.scale, padding_idx=self.padding_idx)


class GroupNormAct(nn.Module):
    """Group norm over the last dimension with a learnt scale and shift, then an activation (``ops.group_norm_act``)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, activation=None):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"{num_channels} channels cannot be divided into {num_groups} groups")
        self.num_groups, self.eps = num_groups, eps
        self.activation = None if activation is None else activation_name(activation)
        self.weight = nn.Parameter(torch.empty(num_channels))
        self.bias = nn.Parameter(torch.empty(num_channels))
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.ones_(self.weight)
        nn.init.zeros_(self.bias)

    def forward(self, x):
        return ops.group_norm_act(x, self.num_groups, self.weight, self.bias, eps=self.eps, activation=self.activation)


def exact_labels(dtype):
    """The numbers of labels, counted from zero, that a floating-point type tells apart (2**24 in float32)."""
    return int(2.0 / torch.finfo(dtype).eps)


def label_indices(labels):
    """Labels as int64.  What is no whole number of the type's exact range - a fraction, NaN, an infinity - becomes -1, a row
    that no table has: cast as it is, 0.9 and -0.5 would be label 0, and NaN whatever the device makes of it."""
    if not labels.is_floating_point():
        return labels.to(torch.int64)
    whole = (labels == labels.floor()) & (labels.abs() < exact_labels(labels.dtype))
    return torch.where(whole, labels, -1.0).to(torch.int64)


class ContextNet(nn.Module):
    """``(n, len(labels) + continuous)`` conditional inputs -> the ``(n, features)`` context of a flow.

    The first ``len(labels)`` columns hold labels, whole numbers in ``[0, labels[k])`` (anything else - a label outside, a
    fraction, NaN - gives a context of NaN, so that the loss shows it), the others continuous values.  Their embeddings and a
    linear map are added, then ``num_layers`` times group norm, activation and a linear layer follow.  Inputs of a type in
    which some labels of a table run together (more than 2**24 in float32) are refused.
    """

    def __init__(self, features, labels=(), continuous=0, hidden_features=32, num_layers=2, num_groups=4,
                 activation="silu"):
        super().__init__()
        self.features, self.labels, self.continuous = int(features), tuple(int(k) for k in labels), int(continuous)
        if self.features < 1 or self.continuous < 0 or any(k < 1 for k in self.labels):
            raise ValueError("features and the numbers of labels must be positive")
        if not self.labels and not self.continuous:
            raise ValueError("a ContextNet needs labels or continuous columns")
        if num_layers < 1:
            raise ValueError("a ContextNet needs at least one layer")
        self.embeddings = nn.ModuleList([Embedding(k, hidden_features) for k in self.labels])
        self.continuous_layer = nn.Linear(self.continuous, hidden_features) if self.continuous else None
        self.norms = nn.ModuleList([GroupNormAct(num_groups, hidden_features, activation=activation)
                                    for _ in range(num_layers)])
        sizes = [hidden_features] * num_layers + [self.features]
        self.layers = nn.ModuleList([nn.Linear(i, o) for i, o in zip(sizes[:-1], sizes[1:])])

    def forward(self, inputs):
        columns = len(self.labels) + self.continuous
        if inputs.dim() != 2 or inputs.shape[1] != columns:
            raise ValueError(f"Expected conditional inputs of shape (N, {columns}), got {tuple(inputs.shape)}")
        if self.continuous and inputs.dtype == torch.float64:
            raise TypeError("ContextNet computes in float32 and casts nothing down silently: the conditional inputs are float64")
        parts = []
        if self.labels:
            if inputs.is_floating_point() and max(self.labels) > exact_labels(inputs.dtype):
                raise ValueError(f"{max(self.labels)} labels cannot be told apart in inputs of type {inputs.dtype}")
            ids = label_indices(inputs[:, : len(self.labels)])
            parts = [embedding(ids[:, k]) for k, embedding in enumerate(self.embeddings)]
        if self.continuous_layer is not None:
            parts.append(self.continuous_layer(inputs[:, len(self.labels) :].to(torch.float32)))
        h = parts[0]
        for part in parts[1:]:
            h = h + part
        for norm, layer in zip(self.norms, self.layers):
            h = layer(norm(h))
        return h


class ContextFlow(BaseFlow):
    """``flow``, a conditional ``HipFlow``, under the context that ``net`` makes of the conditional inputs; the two train
    together.  Every method takes the conditional inputs as ``context``."""

    def __init__(self, flow, net):
        super().__init__()
        if not isinstance(flow, HipFlow) or not flow.context_features:
            raise TypeError("a ContextFlow needs a conditional nessai_amd flow (context_features)")
        if getattr(net, "features", flow.context_features) != flow.context_features:
            raise ValueError(f"the net makes {net.features} context features, the flow takes {flow.context_features}")
        self.flow, self.net = flow, net

    def to(self, device):
        super().to(device)
        self.flow.device = self.device

    def _context(self, context):
        if context is None:
            raise ValueError("a ContextFlow needs its conditional inputs (context)")
        if not isinstance(context, torch.Tensor) or context.device.type != "cuda":
            raise RuntimeError("nessai_amd flows take tensors on a ROCm device; there is no CPU fallback")
        return self.net(context)

    def _fixed(self, context):
        """The context of the directions that autograd does not record (inverse, samples)."""
        with torch.no_grad():
            return self._context(context)

    def _forward(self, x, mode, context, want_x=True):
        z, out, _ = self.flow._run(x, DIR_FORWARD, mode, want_x=want_x, context=self._context(context),
                                   context_trained=True)
        return z, out

    def forward(self, x, context=None):
        return self._forward(x, MODE_APPLY, context)

    def log_prob(self, x, context=None):
        return self._forward(x, MODE_LOGPROB, context, want_x=False)[1]

    def forward_and_log_prob(self, x, context=None):
        return self._forward(x, MODE_LOGPROB, context)

    def inverse(self, z, context=None):
        return self.flow.inverse(z, context=self._fixed(context))

    def sample(self, n, context=None):
        return self.flow.sample(n, context=self._fixed(context))

    def sample_and_log_prob(self, n, context=None):
        return self.flow.sample_and_log_prob(n, context=self._fixed(context))

    def sample_latent_distribution(self, n, context=None):
        return self.flow.sample_latent_distribution(n)

    def base_distribution_log_prob(self, z, context=None):
        return self.flow.base_distribution_log_prob(z)

    def freeze_transform(self):
        self.flow.freeze_transform()

    def unfreeze_transform(self):
        self.flow.unfreeze_transform()


def build_context_net(spec):
    """The net of ``flow_config["context_net"]``: a module with a ``features`` attribute, or ``ContextNet``'s arguments."""
    if isinstance(spec, dict):
        return ContextNet(**spec)
    if isinstance(spec, nn.Module) and hasattr(spec, "features"):
        return spec
    raise TypeError("context_net must be a dictionary of ContextNet's arguments or a module with a `features` attribute")
