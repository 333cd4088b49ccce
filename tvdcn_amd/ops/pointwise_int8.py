"""The pointwise convolution in 8 bits, for inference: ``quantize_int8``, ``dequantize_int8``, ``pointwise_conv_int8``,
``PointwiseConvInt8``.

Maps have one scale per pixel and weights one per output channel, so the products are of whole numbers and the scales
are applied to their sums. No counterpart in the reference.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from ..extension import _assert_has_ops
from ..utils import _activation_code, _log_api_usage_once
from .pointwise import PointwiseConv

__all__ = ["quantize_int8", "dequantize_int8", "pointwise_conv_int8", "PointwiseConvInt8"]


def quantize_int8(input: Tensor) -> Tuple[Tensor, Tensor]:
    r"""A (batch, channels, \*size) map in 8 bits: int8 codes of its shape, channels-last, and a float32 scale for every
    pixel, (batch, \*size). A weight (out_channels, in_channels) has a scale for every output channel so.

    ``scale = max(max |x| * (1 / 127), 2**-126)``, the product in float32 with 1 / 127 rounded to it (at most the last bit
    off the rounded quotient), at most the largest scale of which 127 are finite. A code is ``x / scale`` rounded to the
    nearest integer, ties to even, as if the quotient were exact. A code stands for ``code * scale``. A pixel that holds an
    infinity or a NaN has the scale NaN. float32, float16 and bfloat16. Not differentiable: a call that would need a gradient
    raises.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(quantize_int8)
    _assert_has_ops()
    return torch.ops.tvdcn.quantize_int8(input)


def dequantize_int8(codes: Tensor, scales: Tensor, dtype: torch.dtype) -> Tensor:
    r"""The (batch, channels, \*size) map ``codes * scales``, rounded to ``dtype``, channels-last. Not
    differentiable: a call that would need a gradient raises."""
    _assert_has_ops()
    return torch.ops.tvdcn.dequantize_int8(codes, scales, dtype)


def pointwise_conv_int8(codes: Tensor, scales: Tensor, weight_codes: Tensor, weight_scales: Tensor,
                        bias: Optional[Tensor] = None, residual: Optional[Tensor] = None, activation: str = "none",
                        dtype: torch.dtype = torch.bfloat16) -> Tensor:
    r"""``activation(weight @ input + bias) + residual`` over the channels of every pixel, of an input and a weight in 8 bits.

    Arguments:
        codes (Tensor[batch, in_channels, \*size]), scales (Tensor[batch, \*size]): the input, from :func:`quantize_int8`
            or :func:`rms_norm_int8`. int8 and float32; channels-last codes are read as they are, others are copied
            first. At most 131071 channels.
        weight_codes (Tensor[out_channels, in_channels]), weight_scales (Tensor[out_channels]): the weight, from
            :func:`quantize_int8`. Both may have more axes of size one, as a convolution's weight has.
        bias (Tensor[out_channels]), residual (Tensor[batch, out_channels, \*size]): of type ``dtype`` (autocast
            rounds them to it).
        activation (str): "none", "relu", "silu" or "gelu" (with the error function).
        dtype: of the result: float32, float16 or bfloat16.

    The products are summed exactly; scales, bias, activation and residual are applied in float32 (the scales in an order
    that overflows only where their result does) and the result is rounded once. Not differentiable: a call that would need
    a gradient raises.

    Returns:
        Tensor[batch, out_channels, \*size]: channels-last.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(pointwise_conv_int8)
    _assert_has_ops()
    if weight_codes.dim() > 2:
        if weight_codes.numel() != weight_codes.size(0) * weight_codes.size(1):
            raise RuntimeError("pointwise_conv_int8: expected weight codes of shape (out_channels, in_channels) and axes of "
                               "size one, got {}".format(list(weight_codes.shape)))
        weight_codes, weight_scales = weight_codes.flatten(1), weight_scales.flatten()
    return torch.ops.tvdcn.pointwise_conv_int8(codes, scales, weight_codes, weight_scales, bias, residual,
                                               _activation_code(activation), dtype)


class PointwiseConvInt8(nn.Module):
    """See :func:`pointwise_conv_int8`. Holds the weight's codes and scales as buffers; made from a layer with float weights
    by :meth:`from_float`. A result has the bias's type (the module's ``dtype`` where there is none)."""

    def __init__(self, in_channels: int, out_channels: int, bias: bool = True, activation: str = "none", device=None,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        if in_channels <= 0 or out_channels <= 0:
            raise ValueError("in_channels and out_channels must be positive")
        _activation_code(activation)
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.activation = activation
        self.dtype = dtype
        self.register_buffer("weight_codes", torch.zeros(out_channels, in_channels, device=device, dtype=torch.int8))
        # (float32 whatever a module's .to(dtype) says: see _apply)
        self.register_buffer("weight_scales", torch.ones(out_channels, device=device, dtype=torch.float32))
        self.register_buffer("bias", torch.zeros(out_channels, device=device, dtype=dtype) if bias else None)

    @classmethod
    def from_float(cls, layer: PointwiseConv, dtype: Optional[torch.dtype] = None) -> "PointwiseConvInt8":
        """``layer``'s weight in 8 bits, for results of type ``dtype`` (its weight's where None)."""
        dtype = layer.weight.dtype if dtype is None else dtype
        made = cls(layer.in_channels, layer.out_channels, layer.bias is not None, layer.activation,
                   layer.weight.device, dtype)
        with torch.no_grad():
            codes, scales = quantize_int8(layer.weight)
            made.weight_codes.copy_(codes)
            made.weight_scales.copy_(scales)
            if made.bias is not None:
                made.bias.copy_(layer.bias)
        return made

    def _apply(self, fn, recurse: bool = True):
        # .half(), .to(dtype) and the like convert floating buffers: the scales move with the others but keep their type
        scales, like = self.weight_scales, torch.empty(0, dtype=self.dtype, device=self.weight_scales.device)
        super()._apply(fn, recurse)
        if self.weight_scales.dtype != torch.float32:
            self.weight_scales = scales.to(self.weight_scales.device)
        self.dtype = fn(like).dtype
        return self

    def forward(self, input: Tensor, scales: Optional[Tensor] = None, residual: Optional[Tensor] = None) -> Tensor:
        """``input``: codes, with their scales, or a map of floating values, which is quantized first."""
        if scales is None:
            input, scales = quantize_int8(input)
        bias = self.bias
        dtype = self.dtype if bias is None else bias.dtype   # (a loaded bias may be of another type than the one it replaces)
        return pointwise_conv_int8(input, scales, self.weight_codes, self.weight_scales, bias, residual, self.activation, dtype)

    def extra_repr(self) -> str:
        s = "{}, {}".format(self.in_channels, self.out_channels)
        if self.bias is None:
            s += ", bias=False"
        if self.activation != "none":
            s += ", activation={}".format(self.activation)
        return s + ", dtype={}".format(self.dtype if self.bias is None else self.bias.dtype)
