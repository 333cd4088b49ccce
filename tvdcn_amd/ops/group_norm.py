"""Group normalisation with an activation on channels-last maps: ``group_norm_act``, ``GroupNormAct``.

What a convolution's output goes through in a model, in one operator with its backward. No
counterpart in the reference.
"""
from typing import Optional

import torch
from torch import Tensor, nn
from torch.nn import init

from ..extension import _assert_has_ops
from ..utils import _activation_code, _log_api_usage_once

__all__ = ["group_norm_act", "GroupNormAct"]


def group_norm_act(input: Tensor, num_groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                   eps: float = 1e-5, activation: str = "none", keep_int8: bool = False) -> Tensor:
    r"""``activation(group_norm(input) * weight + bias)``.

    The mean and the (biased) variance are taken over the pixels and the channels / num_groups channels of each image
    and group, in float32 (float64 for float64 maps, on the CPU only), and the result is rounded once.

    Arguments:
        input (Tensor[batch, channels, \*size]): the map; channels-last memory (``torch.channels_last`` in 2D) is read
            as it is, any other is copied first. (rows, channels) is a map without a grid.
        num_groups (int): divides the channels.
        weight, bias (Tensor[channels]): of the input's type (autocast rounds them to it); 1 and 0 where absent.
        eps (float): added to the variance.
        activation (str): "none", "relu", "silu" or "gelu" (with the error function).
        keep_int8 (bool): the input is kept for the backward in 8 bits (see :func:`compress_activation`), and the
            backward takes the gradients at the values kept. The output does not change.

    Returns:
        Tensor[batch, channels, \*size]: channels-last. First derivatives by backward only: second ones and forward-mode
        ones raise.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(group_norm_act)
    _assert_has_ops()
    return torch.ops.tvdcn.group_norm_act(input, num_groups, weight, bias, eps, _activation_code(activation), keep_int8)


class GroupNormAct(nn.Module):
    """See :func:`group_norm_act`."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "none", keep_int8: bool = False, device=None, dtype=None) -> None:
        super().__init__()
        if num_groups <= 0 or num_channels % num_groups != 0:
            raise ValueError("num_channels must be divisible by num_groups")
        _activation_code(activation)
        self.num_groups = num_groups
        self.num_channels = num_channels
        self.eps = float(eps)
        self.affine = affine
        self.activation = activation
        self.keep_int8 = keep_int8
        if affine:
            self.weight = nn.Parameter(torch.empty(num_channels, device=device, dtype=dtype))
            self.bias = nn.Parameter(torch.empty(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        if self.affine:
            init.ones_(self.weight)
            init.zeros_(self.bias)

    def forward(self, input: Tensor) -> Tensor:
        return group_norm_act(input, self.num_groups, self.weight, self.bias, self.eps, self.activation, self.keep_int8)

    def extra_repr(self) -> str:
        s = "{}, {}, eps={}, affine={}".format(self.num_groups, self.num_channels, self.eps, self.affine)
        if self.activation != "none":
            s += ", activation={}".format(self.activation)
        return s + (", keep_int8=True" if self.keep_int8 else "")
