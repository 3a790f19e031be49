"""The dense layers around a forest as functions: a gated projection in front of one, the loss of a linear layer's class scores
behind one.

The reference has neither as an operator: its pipelines put torch.nn modules in front of a forest and take the loss of the scores that
a (fused) linear layer writes (README.md:110-129).
"""
from .._ext import hingetree_cpp


def gated_linear(x, gate_weight, value_weight, gate_bias=None, value_bias=None, activation="silu"):
    """act(x @ gate_weight.T + gate_bias) * (x @ value_weight.T + value_bias), both projections, the activation and the product in
    one kernel.

    x: [..., features]; weights: [outputs, features]; biases: [outputs] or None; all torch.float32, bfloat16 or float16, one type for all.
    activation: 'silu', 'gelu' (with the normal distribution function), 'relu' or 'sigmoid'.  Sums are fp32 whatever the type, and
    fp32 results are as accurate as fp32 products (of finite numbers: an infinity gives NaN, in fp16 gradients too).  The gradients of the two
    projections enter the sums of the backward as bf16 numbers for bfloat16 and as two of them for float16.  The backward forms the
    projections again; of the forward it keeps the inputs and, for fp32 and for 16-bit rows that do not start on 16 bytes, their copies in the tensor
    cores' layout (6 or 2 bytes a number; hingetree_cpp.set_save_forward(False): none).  No second derivative."""
    return hingetree_cpp.gated_linear(x, gate_weight, value_weight, gate_bias, value_bias, activation)


def linear_class_loss(x, weight, bias, target, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of the class scores x @ weight.T + bias, which never lie in memory, and its gradient.

    x: [..., features]; weight: [classes, features]; bias: [classes] or None; one type of torch.float32, bfloat16 or float16 for all;
    target: int64, [...].  The loss is float32 whatever the type: one number for 'mean' (over the rows that count; NaN where none
    does) and 'sum', one per row for 'none'.

    For 16-bit types the scores are summed in the tensor cores, which truncate: a loss is off by about 3e-7 of its size at 1000 features.  The
    backward holds the gradient of the scores as gated_linear's holds that of its projections.

    A row whose target is ignore_index has loss and gradient 0 whatever it holds.  A target that is neither a class nor ignore_index
    makes the loss NaN, and the next hingetree_cpp.pipeline_status() raises RuntimeError.  The backward holds the gradient of the scores
    in pieces of 512 MiB at the most, less with hingetree_cpp.set_backward_scratch_limit(bytes), and what gated_linear keeps of its inputs.  No second derivative."""
    return hingetree_cpp.linear_class_loss(x, weight, bias, target, ignore_index, reduction)
