"""The dense layers around a forest as modules: GatedLinear, a gated projection whose results are a forest's features, and
LinearClassLoss, a linear layer behind one that gives the loss instead of the class scores.

The reference's pipelines put torch.nn modules in front of a forest and take a loss of written scores (README.md:110-129).
"""
import math

import torch
import torch.nn as nn

from .. import HingeTree as _F
from ._Answers import PackedClasses


def _linear_parameters(outputs, inputs, bias):
    """Weight and bias as nn.Linear initialises them."""
    weight = nn.Parameter(torch.empty(outputs, inputs))
    nn.init.kaiming_uniform_(weight, a=math.sqrt(5))
    if not bias:
        return weight, None
    bound = 1 / math.sqrt(inputs) if inputs > 0 else 0
    return weight, nn.Parameter(torch.empty(outputs).uniform_(-bound, bound))


class GatedLinear(nn.Module):
    """act(gate(x)) * value(x) with two linear layers, in one kernel: features for a forest.  x: [..., in_features]; parameters
    ``gate_weight``, ``value_weight`` [out_features, in_features] and, with bias, ``gate_bias``, ``value_bias``.  activation: 'silu',
    'gelu', 'relu' or 'sigmoid'.  float32, bfloat16 or float16, as its parameters are."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "silu"):
        super().__init__()
        if activation not in ("silu", "gelu", "relu", "sigmoid"):
            raise ValueError("activation must be 'silu', 'gelu', 'relu' or 'sigmoid'")
        self.in_features, self.out_features, self.activation = in_features, out_features, activation
        self.gate_weight, self.gate_bias = _linear_parameters(out_features, in_features, bias)
        self.value_weight, self.value_bias = _linear_parameters(out_features, in_features, bias)

    def forward(self, x):
        return _F.gated_linear(x, self.gate_weight, self.value_weight, self.gate_bias, self.value_bias, self.activation)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, bias=%s, activation=%s" % (self.in_features, self.out_features,
                                                                            self.gate_bias is not None, self.activation)


class LinearClassLoss(nn.Module):
    """Softmax cross entropy of linear class scores that never lie in memory: nn.Linear followed by nn.CrossEntropyLoss, with
    nn.Linear's parameters ``weight`` [classes, in_features] and ``bias``.  forward(x, target) gives the loss (float32); scores(x) gives
    the class scores, for answers."""

    def __init__(self, in_features: int, classes: int, bias: bool = True, ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        if reduction not in ("none", "mean", "sum"):
            raise ValueError("reduction must be 'none', 'mean' or 'sum'")
        self.in_features, self.classes, self.ignore_index, self.reduction = in_features, classes, ignore_index, reduction
        self.weight, self.bias = _linear_parameters(classes, in_features, bias)

    def forward(self, x, target):
        return _F.linear_class_loss(x, self.weight, self.bias, target, self.ignore_index, self.reduction)

    def scores(self, x):
        return nn.functional.linear(x, self.weight, self.bias)

    @torch.no_grad()
    def sample(self, x, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """A class drawn from the scores of each row, and the logarithm of its share (HingeTree.sample_classes)."""
        return _F.sample_classes(self.scores(x), uniform, temperature, top_k, top_p, min_p)

    def packed(self):
        """The same scores under weights in 4 bits, for answers (PackedClasses)."""
        return PackedClasses.of(self.weight, self.bias)

    def extra_repr(self):
        return "in_features=%d, classes=%d, bias=%s, ignore_index=%d, reduction=%s" % (
            self.in_features, self.classes, self.bias is not None, self.ignore_index, self.reduction)
