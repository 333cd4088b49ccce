"""The pointwise convolution with bias, activation and residual: ``pointwise_conv``, ``PointwiseConv``.

A matrix product over the channels of every pixel (a 1x1 convolution, or a linear layer over the rows of a
matrix), with what follows it in a block applied as its results are written. No counterpart in the
reference.
"""
import math
from typing import Optional

import torch
from torch import Tensor, nn
from torch.nn import init

from ..extension import _assert_has_ops
from ..utils import _activation_code, _log_api_usage_once

__all__ = ["pointwise_conv", "PointwiseConv"]


def pointwise_conv(input: Tensor, weight: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None,
                   activation: str = "none", keep_int8: bool = False) -> Tensor:
    r"""``activation(weight @ input + bias) + residual`` over the channels of every pixel.

    Arguments:
        input (Tensor[batch, in_channels, \*size]): the map; channels-last memory (``torch.channels_last`` in 2D) is
            read as it is, any other is copied first. (rows, in_channels) is a map without a grid.
        weight (Tensor[out_channels, in_channels]): may have more axes of size one, as a convolution's has.
        bias (Tensor[out_channels]), residual (Tensor[batch, out_channels, \*size]): of the input's type.
        activation (str): "none", "relu", "silu" or "gelu" (with the error function).
        keep_int8 (bool): the input is kept for the weight's gradient in 8 bits (see :func:`compress_activation`),
            which is taken with the values kept. The output and the other gradients do not change.

    Values are multiplied as they are and summed in float32 (large float32 products as three bfloat16 pieces per value,
    to the same precision; an infinite value may give a NaN there); the result is rounded once. The backward reads the
    activation's argument, kept in the input's type (float16 for "silu" and "gelu" of bfloat16), and rounds its gradient
    to the input's type before the products. float64 runs on the CPU only.

    Returns:
        Tensor[batch, out_channels, \*size]: channels-last. First derivatives by backward only: second ones and forward-mode
        ones raise.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(pointwise_conv)
    _assert_has_ops()
    if weight.dim() > 2:
        if weight.numel() != weight.size(0) * weight.size(1):
            raise RuntimeError("pointwise_conv: expected a weight of shape (out_channels, in_channels) and axes of size "
                               "one, got {}".format(list(weight.shape)))
        weight = weight.flatten(1)
    return torch.ops.tvdcn.pointwise_conv(input, weight, bias, residual, _activation_code(activation), keep_int8)


class PointwiseConv(nn.Module):
    """See :func:`pointwise_conv`."""

    def __init__(self, in_channels: int, out_channels: int, bias: bool = True, activation: str = "none",
                 keep_int8: bool = False, device=None, dtype=None) -> None:
        super().__init__()
        if in_channels <= 0 or out_channels <= 0:
            raise ValueError("in_channels and out_channels must be positive")
        _activation_code(activation)
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.activation = activation
        self.keep_int8 = keep_int8
        self.weight = nn.Parameter(torch.empty(out_channels, in_channels, device=device, dtype=dtype))
        if bias:
            self.bias = nn.Parameter(torch.empty(out_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        bound = 1 / math.sqrt(self.in_channels)
        init.uniform_(self.weight, -bound, bound)
        if self.bias is not None:
            init.uniform_(self.bias, -bound, bound)

    def forward(self, input: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        return pointwise_conv(input, self.weight, self.bias, residual, self.activation, self.keep_int8)

    def extra_repr(self) -> str:
        s = "{}, {}".format(self.in_channels, self.out_channels)
        if self.bias is None:
            s += ", bias=False"
        if self.activation != "none":
            s += ", activation={}".format(self.activation)
        return s + (", keep_int8=True" if self.keep_int8 else "")
