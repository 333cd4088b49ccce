"""Root-mean-square normalisation of every pixel's channels: ``rms_norm``, ``add_rms_norm`` (with the shortcut's addition),
their 8-bit forms for inference, ``RMSNorm`` and ``AddRMSNorm``.

A pixel is one token: nothing is averaged over the grid. No counterpart in the reference.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor, nn
from torch.nn import init

from ..extension import _assert_has_ops
from ..utils import _log_api_usage_once

__all__ = ["rms_norm", "add_rms_norm", "rms_norm_int8", "add_rms_norm_int8", "RMSNorm", "AddRMSNorm"]


def rms_norm(input: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6) -> Tensor:
    r"""``weight * input / sqrt(mean(input**2) + eps)``, the mean over the channels of every pixel.

    Arguments:
        input (Tensor[batch, channels, \*size]): the map; channels-last memory (``torch.channels_last`` in 2D) is read
            as it is, any other is copied first. (rows, channels) is a map without a grid.
        weight (Tensor[channels]): of the input's type (autocast rounds it to that); 1 where absent.
        eps (float): added to the mean; a normal float32 above zero.

    Sums are held in float32 (float64 for float64 maps, on the CPU only) and the result is rounded once. A pixel that holds
    an infinity or a NaN has zeros and NaN, as the formula has.

    Returns:
        Tensor[batch, channels, \*size]: channels-last. First derivatives by backward only: second ones and forward-mode
        ones raise.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(rms_norm)
    _assert_has_ops()
    return torch.ops.tvdcn.rms_norm(input, weight, eps)


def add_rms_norm(input: Tensor, residual: Tensor, weight: Optional[Tensor] = None,
                 eps: float = 1e-6) -> Tuple[Tensor, Tensor]:
    r""":func:`rms_norm` of ``input + residual``, and that sum, both in one pass over the maps.

    The sum is rounded to the maps' type and normalised as rounded. ``residual`` has the input's shape and type (under
    autocast both take the wider one of their types).

    Returns:
        (Tensor, Tensor): the normalised map and the sum, channels-last, both differentiable as :func:`rms_norm` is.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(add_rms_norm)
    _assert_has_ops()
    return torch.ops.tvdcn.add_rms_norm(input, residual, weight, eps)


def rms_norm_int8(input: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6) -> Tuple[Tensor, Tensor]:
    r""":func:`rms_norm` with its result in 8 bits, as :func:`pointwise_conv_int8` reads it.

    The codes and scales are :func:`quantize_int8`'s of the result before it is rounded to the map's type. float32,
    float16 and bfloat16 maps. Not differentiable: a call that would need a gradient raises.

    Returns:
        (Tensor, Tensor): int8 codes of the input's shape, channels-last, and float32 scales (batch, \*size).
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(rms_norm_int8)
    _assert_has_ops()
    return torch.ops.tvdcn.rms_norm_int8(input, weight, eps)


def add_rms_norm_int8(input: Tensor, residual: Tensor, weight: Optional[Tensor] = None,
                      eps: float = 1e-6) -> Tuple[Tensor, Tensor, Tensor]:
    r""":func:`rms_norm_int8` of ``input + residual`` (see :func:`add_rms_norm`).

    Returns:
        (Tensor, Tensor, Tensor): the codes, the scales and the sum, which has the maps' type.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(add_rms_norm_int8)
    _assert_has_ops()
    return torch.ops.tvdcn.add_rms_norm_int8(input, residual, weight, eps)


class RMSNorm(nn.Module):
    """See :func:`rms_norm`."""

    def __init__(self, num_channels: int, eps: float = 1e-6, affine: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        if num_channels <= 0:
            raise ValueError("num_channels must be positive")
        self.num_channels = num_channels
        self.eps = float(eps)
        self.affine = affine
        if affine:
            self.weight = nn.Parameter(torch.empty(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        if self.affine:
            init.ones_(self.weight)

    def forward(self, input: Tensor) -> Tensor:
        return rms_norm(input, self.weight, self.eps)

    def extra_repr(self) -> str:
        return "{}, eps={}, affine={}".format(self.num_channels, self.eps, self.affine)


class AddRMSNorm(RMSNorm):
    """See :func:`add_rms_norm`."""

    def forward(self, input: Tensor, residual: Tensor) -> Tuple[Tensor, Tensor]:
        return add_rms_norm(input, residual, self.weight, self.eps)
