"""8-bit activations: ``compress_activation``, ``expand_activation``.

A feature map held in about a quarter (float32) or a half (16-bit types) of its memory, for what a
model keeps between its forward and its backward. :func:`group_norm_act` and :func:`pointwise_conv`
keep their input so with ``keep_int8=True``. No counterpart in the reference.
"""
from typing import Tuple

import torch
from torch import Tensor

from ..extension import _assert_has_ops

__all__ = ["compress_activation", "expand_activation"]


def compress_activation(input: Tensor) -> Tuple[Tensor, Tensor]:
    r"""The 8-bit form of a (batch, channels, \*size) map: int8 codes of the map's shape and uint8 exponents of
    shape (batch, ceil(channels / 32), \*size), both channels-last.

    Every 32 channels of a pixel share an exponent k, stored as k + 127: the least k >= -126 with
    ``max |x| <= 127 * 2**k``. A code is ``x / 2**k`` rounded to the nearest integer, ties to even, and stands
    for ``code * 2**k``: at most half of ``2**k`` off, that is at most 1/127 of the block's largest value. A block that
    holds an infinity or a NaN comes back as NaN. float32, float16 and bfloat16 maps. Not differentiable.
    """
    _assert_has_ops()
    return torch.ops.tvdcn.compress_activation(input)


def expand_activation(codes: Tensor, exponents: Tensor, dtype: torch.dtype) -> Tensor:
    r"""The (batch, channels, \*size) map of type ``dtype`` that :func:`compress_activation`'s result stands for,
    channels-last. Values are clamped to the finite values of ``dtype``, which is the type of the map that was
    compressed. Not differentiable."""
    _assert_has_ops()
    return torch.ops.tvdcn.expand_activation(codes, exponents, dtype)
