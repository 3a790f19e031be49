"""Answers of a linear layer with many classes as functions: its weights as microscaled 4-bit numbers, class scores under them, and a
class drawn from a row of scores.

The reference has none of them as an operator: its pipelines put torch.nn modules behind a forest (README.md:110-129).
"""
import torch

from .._ext import hingetree_cpp


def pack_mx4(weight):
    """weight [outputs, features] (torch.float32, bfloat16 or float16) as MXFP4 of the Microscaling Formats specification v1.0: (codes, scales),
    both torch.uint8, 17 bytes for 32 features.

    With blocks = features / 32, rounded up: scales [outputs, blocks], byte b for 2 ** (b - 127), the power of two that is 4 times below the one of
    the block's largest magnitude; codes [outputs, 16 * blocks], two to a byte, the first in the low half, each a sign and one of 0, 0.5, 1, 1.5,
    2, 3, 4, 6: the nearest (of two as near the one whose code is even), 6 at the most.  A block with an infinity or NaN stands for NaN.  Takes
    weights that require a gradient; the result has none."""
    codes, scales = hingetree_cpp.pack_mx4(weight)
    return codes, scales


def unpack_mx4(codes, scales, features, dtype=torch.float32):
    """The values [outputs, features] of packed weights; exact in torch.float32 and bfloat16 (those beyond their range
    are infinite), rounded to float16."""
    return hingetree_cpp.unpack_mx4(codes, scales, features, dtype)


def linear_mx4(x, codes, scales, bias=None):
    """x @ W.T + bias with W the values of packed weights, which are read as they are packed.

    x: [..., features], torch.float32, bfloat16 or float16; bias: [outputs] in x's type, or None; the result is in x's type.  Sums are fp32, and
    x enters them exactly: fp32 results are as accurate as fp32 products with the values (of finite numbers: an infinity gives NaN in fp32
    and fp16; of fp32 numbers below 2 ** -110 what is less than 2 ** -134 is lost).  Those of 16-bit x are the tensor core's, which truncates when it adds:
    some 3e-8 of a sum for every 16 features, below a step of the type up to 10 ** 5 of them.  Large calls of bfloat16 (1024 rows and 10 ** 10 multiplications on) hold decoded weights while they run, 2 bytes each and
    512 MiB at the most, or none, at a fifth more time, where memory is short.  No
    derivative: tensors that require a gradient are refused while gradients are recorded."""
    return hingetree_cpp.linear_mx4(x, codes, scales, bias)


def sample_classes(scores, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A class drawn from each row of scores, and the logarithm of its share: (classes int64, log_probs float32), both [...].

    scores: [..., classes], torch.float32, bfloat16 or float16; uniform: torch.float32, [...], numbers in [0, 1].  Each of the bounds is one number, or a
    tensor [...] with one a row (torch.float32; top_k torch.int64).

    A class weighs exp((score - largest) / temperature); with temperature 0 the first class of the largest score is taken.  In the order of
    falling scores, of equal ones the lower class first, the shortest of these prefixes counts, its first class always: top_k classes (0: all); the
    shortest that holds top_p of the weight of the first top_k (1: all of them); the classes that weigh at least min_p.  Of those the
    first is taken, in the order of classes, up to which they weigh more than `uniform` of all of them.  Weights and sums are held in 64
    bits, so that the choice is that of the formula.

    A row without an answer has class -1 and log_prob NaN: its largest score is not finite (all classes masked with -inf among them), a score or
    a bound is NaN, its temperature is negative or infinite, its random number outside [0, 1].  No derivative."""
    classes, log_probs = hingetree_cpp.sample_classes(scores, uniform, temperature, top_k, top_p, min_p)
    return classes, log_probs
