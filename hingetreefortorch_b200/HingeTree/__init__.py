"""Autograd functions of the hinge tree drop-in (same exported names as the reference package, plus the dense
layers around a forest)."""
from ._HingeTree import (  # noqa: F401
    contract, expand, Contract, Expand,
    HingeTree, HingeFern, SparseHingeTree, SparseHingeFern,
    HingeTreeFusedLinear, HingeFernFusedLinear, SparseHingeTreeFusedLinear, SparseHingeFernFusedLinear,
    HingeTreeFusion, HingeFernFusion, HingeTreeFusionFusedLinear, HingeFernFusionFusedLinear,
    HingeTreeConv1d, HingeTreeConv2d, HingeTreeConv3d, HingeFernConv1d, HingeFernConv2d, HingeFernConv3d,
    HingeTrie,
)
from ._Dense import gated_linear, linear_class_loss  # noqa: F401
