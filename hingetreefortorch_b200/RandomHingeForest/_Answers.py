"""Answers of a linear layer with many classes as a module: PackedClasses, class scores under weights held as microscaled 4-bit numbers,
and classes drawn from them.

The reference's pipelines put torch.nn modules behind a forest (README.md:110-129).
"""
import torch
import torch.nn as nn

from .. import HingeTree as _F


class PackedClasses(nn.Module):
    """A class head for answers: nn.Linear whose weight is held as 4-bit numbers with a power of two for each 32 features
    (HingeTree.pack_mx4), 17 bytes for 32 of them.  Buffers ``codes``, ``scales`` (uint8) and, with bias, ``bias``; no parameters, no derivative.
    x: [..., in_features] in the bias's type (without one: torch.float32, bfloat16 or float16); forward(x) gives the class scores (x that requires a
    gradient is refused while gradients are recorded), sample(x, uniform, ...) a class drawn from them and the logarithm of its share
    (HingeTree.sample_classes), without a gradient whatever x requires.

    PackedClasses.of(weight, bias) packs a layer's; LinearClassLoss.packed() and RandomHingeForestFusedLinear.packed_classes() give theirs."""

    def __init__(self, in_features: int, classes: int, bias: bool = True):
        super().__init__()
        self.in_features, self.classes = in_features, classes
        blocks = -(-in_features // 32)
        self.register_buffer("codes", torch.zeros(classes, 16 * blocks, dtype=torch.uint8))
        self.register_buffer("scales", torch.zeros(classes, blocks, dtype=torch.uint8))
        self.register_buffer("bias", torch.zeros(classes) if bias else None)

    @classmethod
    def of(cls, weight, bias=None):
        classes, in_features = weight.shape
        head = cls(1, 1, bias is not None)
        head.in_features, head.classes = in_features, classes
        head.codes, head.scales = _F.pack_mx4(weight)
        if bias is not None:
            head.bias = bias.detach().clone()
        return head

    def forward(self, x):
        return _F.linear_mx4(x, self.codes, self.scales, self.bias)

    scores = forward

    @torch.no_grad()
    def sample(self, x, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        return _F.sample_classes(self(x), uniform, temperature, top_k, top_p, min_p)

    def extra_repr(self):
        return "in_features=%d, classes=%d, bias=%s" % (self.in_features, self.classes, self.bias is not None)
