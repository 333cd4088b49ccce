"""Dropout whose mask is never stored: ``seeded_dropout``, ``SeededDropout``.

The mask follows from a seed and a value's place, so the backward makes it again. No counterpart in the reference.
"""
from typing import Optional

import torch
from torch import Tensor, nn

from ..extension import _assert_has_ops
from ..utils import _log_api_usage_once

__all__ = ["seeded_dropout", "SeededDropout"]


def _draw_seed(input: Tensor) -> Tensor:
    return torch.randint(0x7FFFFFFFFFFFFFFF, [1], dtype=torch.int64, device=input.device)


def seeded_dropout(input: Tensor, p: float, seed: Optional[Tensor] = None, residual: Optional[Tensor] = None) -> Tensor:
    r"""Every value of the map dropped (zero) with probability p, the others divided by 1 - p, plus ``residual``.

    Arguments:
        input (Tensor[batch, channels, \*size]): the map; channels-last memory (``torch.channels_last`` in 2D) is read
            as it is, any other is copied first. (rows, channels) is a map without a grid.
        p (float): in [0, 1], taken as the nearest multiple of 2**-16.
        seed (Tensor): one int64 on the input's device; drawn from torch's generator of that device where None. The
            same seed gives the same mask for maps of the same shape, whatever their type, memory order or device. It is
            read when the kernels run: in a captured graph, writing to it gives the next replay another mask (do
            so between steps, not between a forward and its backward).
        residual (Tensor[batch, channels, \*size]): of the input's type (under autocast both take the wider one of
            their types).

    The bits are Philox4x32-10's (Salmon et al., 2011), keyed by the seed and counted along the map's channels-last memory, 16
    bits a value. The scaling and the sum are float32 and rounded once; a dropped value is zero whatever it holds.

    Returns:
        Tensor[batch, channels, \*size]: channels-last. Derivatives by backward only: forward-mode ones raise.
    """
    if not torch.jit.is_scripting():
        _log_api_usage_once(seeded_dropout)
    _assert_has_ops()
    if seed is None:
        seed = _draw_seed(input)
    return torch.ops.tvdcn.seeded_dropout(input, p, seed, residual)


class SeededDropout(nn.Module):
    """See :func:`seeded_dropout`. In training every call draws a seed; in evaluation nothing is dropped."""

    def __init__(self, p: float = 0.5) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("p must be in [0, 1], got {}".format(p))
        self.p = p

    def forward(self, input: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        if self.training:
            return seeded_dropout(input, self.p, None, residual)
        return input if residual is None else input + residual

    def extra_repr(self) -> str:
        return "p={}".format(self.p)
