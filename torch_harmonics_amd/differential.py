"""
DifferentialNeighborhoodAttentionS2: neighborhood attention whose output is the difference of two softmax maps with a learned weight per
head, normed per head; and GroupNormS2, the group norm over the sphere that it uses.
"""

import math
from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
import torch.nn.functional as F

from ._attention_utils import _check_extent, _check_ndim
from ._layout import to_nchw, to_nhwc
from ._lib import ACTIVATIONS
from .attention import NeighborhoodAttentionS2
from .ops import differential_s2_attention, group_norm_s2
from .quadrature import precompute_latitudes

__all__ = ["DifferentialNeighborhoodAttentionS2", "GroupNormS2"]


def _ring_weights(nlat: int, nlon: int, grid: str) -> torch.Tensor:
    """Quadrature weight of a point on each latitude ring; the rings sum to 4 pi."""
    _, w = precompute_latitudes(nlat, grid=grid)
    return (2.0 * torch.pi * w.to(dtype=torch.float32) / nlon).contiguous()


class GroupNormS2(nn.Module):
    r"""
    Group norm over the sphere with an activation: mean and variance of every group of channels over the grid, weighted by the grid's
    quadrature, so that the crowded rings at the poles count by their area.

    Parameters
    ----------
    num_groups, num_channels : int
        groups must divide channels
    shape : (nlat, nlon), optional
        the grid; without it every point counts the same, on any grid
    grid : str
        ``"equiangular"``, ``"legendre-gauss"``, ``"lobatto"`` or ``"equiangular-trapezoidal"``
    eps : float
        added to the variance
    affine : bool
        learnable weight and bias per channel
    activation : str, optional
        ``"relu"``, ``"silu"`` or ``"gelu"``, applied to the result
    """

    def __init__(
        self,
        num_groups: int,
        num_channels: int,
        shape: Optional[Tuple[int]] = None,
        grid: Optional[str] = "equiangular",
        eps: Optional[float] = 1e-5,
        affine: Optional[bool] = True,
        activation: Optional[str] = None,
    ):
        super().__init__()
        if num_channels % num_groups != 0:
            raise ValueError(f"Please make sure that number of groups {num_groups} divides num_channels {num_channels} evenly.")
        if activation is not None and activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}, or None")
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        self.shape = None if shape is None else tuple(shape)
        self.register_buffer("quad_weights", None if shape is None else _ring_weights(*shape, grid), persistent=False)
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def extra_repr(self):
        return f"num_groups={self.num_groups}, num_channels={self.num_channels}, shape={self.shape}, activation={self.activation}"

    def forward_nhwc(self, x: torch.Tensor) -> torch.Tensor:
        """(B, nlat, nlon, num_channels) -> the same."""
        return group_norm_s2(x, self.num_groups, self.weight, self.bias, self.quad_weights, self.eps, self.activation)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """(B, num_channels, nlat, nlon) -> the same, in the memory format of x (channels last, or channels first)."""
        _check_ndim(x, 4, "input")
        _check_extent(x, 1, self.num_channels, "input channels")
        if self.shape is not None:
            _check_extent(x, -2, self.shape[0], "input latitudes")
            _check_extent(x, -1, self.shape[1], "input longitudes")
        if x.is_contiguous(memory_format=torch.channels_last):
            return self.forward_nhwc(x.permute(0, 2, 3, 1)).permute(0, 3, 1, 2)
        return to_nchw(self.forward_nhwc(to_nhwc(x)))


class DifferentialNeighborhoodAttentionS2(NeighborhoodAttentionS2):
    r"""
    Differential neighborhood attention on the 2-sphere: each head has two query and two key vectors, and its output is

    .. math:: y = \sum_j (p^1_j - \lambda p^2_j) v_j, \qquad \lambda = e^{\lambda_{q1} \cdot \lambda_{k1}} - e^{\lambda_{q2} \cdot \lambda_{k2}} + \lambda_\mathrm{init}

    with :math:`p^1, p^2` the quadrature-weighted softmaxes over the points inside the disk around the output point.  The difference
    takes off what both maps give to everything in the disk.  The output is normed head by head, times :math:`1 - \lambda_\mathrm{init}`.

    Parameters are those of NeighborhoodAttentionS2, with the same projections (a head's ``k_channels // num_heads`` channels of q and k are
    two vectors of half as many), and

    Parameters
    ----------
    scale : float or Tensor, optional
        multiplies the query; default ``1 / sqrt(k_channels // (2 * num_heads))``
    use_qknorm : bool
        RMS normalisation of each of the two vectors, with learnable gain ``1 + w``
    lambda_init : float
        the learned weight's constant part
    norm : str, optional
        ``"group"``: group norm over the grid with a head's channels as a group, weighted by the output grid's quadrature, learnable weight and
        bias; ``"rms"``: per point and head, learnable gain ``1 + w``; None
    activation : str, optional
        ``"relu"``, ``"silu"`` or ``"gelu"`` on the result of the group norm
    """

    def __init__(
        self,
        in_channels: int,
        in_shape: Tuple[int],
        out_shape: Tuple[int],
        grid_in: Optional[str] = "equiangular",
        grid_out: Optional[str] = "equiangular",
        num_heads: Optional[int] = 1,
        scale: Optional[Union[torch.Tensor, float]] = None,
        use_qknorm: Optional[bool] = False,
        bias: Optional[bool] = True,
        theta_cutoff: Optional[float] = None,
        k_channels: Optional[int] = None,
        out_channels: Optional[int] = None,
        optimized_kernel: Optional[bool] = True,
        lambda_init: Optional[float] = 0.8,
        norm: Optional[str] = "group",
        activation: Optional[str] = None,
    ):
        if norm not in ("group", "rms", None):
            raise ValueError(f"unknown norm {norm!r}: 'group', 'rms' or None")
        if activation is not None and norm != "group":
            raise ValueError("an activation is part of the group norm: it needs norm='group'")
        width = in_channels if k_channels is None else k_channels
        if width % (2 * num_heads) != 0:
            raise ValueError(f"Please make sure that twice the number of heads {num_heads} divides k_channels {width} evenly: two maps per head.")
        ck = width // (2 * num_heads)
        super().__init__(
            in_channels, in_shape, out_shape, grid_in, grid_out, num_heads, scale if scale is not None else 1 / math.sqrt(ck), use_qknorm, bias, theta_cutoff, k_channels, out_channels,
            optimized_kernel,
        )  # fmt: skip
        if use_qknorm:
            self.q_norm_weights = nn.Parameter(torch.zeros(ck))
            self.k_norm_weights = nn.Parameter(torch.zeros(ck))
        self.lambda_init = lambda_init
        for name in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2"):
            setattr(self, name, nn.Parameter(0.1 * torch.randn(num_heads, ck)))
        self.norm, self.activation = norm, activation
        if norm == "group":
            self.head_norm = GroupNormS2(num_heads, self.out_channels, out_shape, grid_out, activation=activation)
        elif norm == "rms":
            self.head_norm_weights = nn.Parameter(torch.zeros(self.out_channels // num_heads))
        self.attention_handle = differential_s2_attention

    def learned_lambda(self) -> torch.Tensor:
        """The weight of the second map, one number per head."""
        one, two = (self.lambda_q1 * self.lambda_k1).sum(-1), (self.lambda_q2 * self.lambda_k2).sum(-1)
        return torch.exp(one) - torch.exp(two) + self.lambda_init

    def _native_dtype(self, query, key, value):
        return None  # composed of separate operators

    def _head_rms_norm(self, x: torch.Tensor, gain: torch.Tensor, scale=None) -> torch.Tensor:
        shape = x.shape
        x = F.rms_norm(x.reshape(*shape[:3], -1, gain.shape[0]), normalized_shape=gain.shape, weight=1 + gain if scale is None else (1 + gain) * scale)
        return x.reshape(shape)

    def _attend_and_project(self, query, key, value, normed: bool, direct: bool) -> torch.Tensor:
        """NHWC q, k, v -> the module's NCHW output."""
        if normed:
            query = self._head_rms_norm(query, self.q_norm_weights, self.scale)
            key = self._head_rms_norm(key, self.k_norm_weights)
        out = self.attention_handle(
            key, value, query, self.learned_lambda(), self.quad_weights, self.psi_col_idx, self.psi_roff_idx, self.num_heads, self.nlon_in, self.nlat_out, self.nlon_out,
            self.psi_plan, self._psi_plan_header,
        )  # fmt: skip
        if self.norm == "group":
            n = self.head_norm
            rest = 1 - self.lambda_init
            if n.activation is None:  # (the factor rides on the parameters: no pass of its own)
                out = group_norm_s2(out, n.num_groups, n.weight * rest, n.bias * rest, n.quad_weights, n.eps)
            else:
                out = n.forward_nhwc(out) * rest
        elif self.norm == "rms":
            out = self._head_rms_norm(out, self.head_norm_weights, 1 - self.lambda_init)
        return self._project(out, direct)
