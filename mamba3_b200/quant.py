"""4-bit projection weights with group scales, for decoding.

A weight ``[out, in]`` is held as ``codes`` (uint8 ``[out, ceil(in / 2)]``, two 4-bit codes to a byte,
the even column in the low half), ``scales`` ``[out, ceil(in / group)]`` and optional ``zeros`` of the
same shape: ``w = scale * (code - zero)``, zero 8 where none is given. :func:`quantize_w4` makes them,
:func:`linear_w4` multiplies with them (``m3_linear_w4`` on CUDA), :class:`LinearW4` stands in for an
``nn.Linear`` without bias, and :func:`quantize_projections` replaces a model's.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.nn import functional as F

from . import _ext

_GROUPS = (32, 64, 128)


def quantize_w4(weight: torch.Tensor, *, group_size: int = 128, zeros: bool = False, dtype: torch.dtype | None = None):
    """``(codes, scales, zeros or None)`` of a ``[out, in]`` weight, rounding to nearest per group.

    Without ``zeros`` a group spans ``[-8, 7] * scale`` with ``scale = max|w| / 7.5`` (codes clamped);
    with them it spans its minimum to its maximum, 0 among them, and the zero point is a
    number in [0, 15]. Scales and zeros are ``dtype`` (the
    weight's by default), and the codes are chosen against the rounded scales.
    """
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError("weight must be a floating-point [out, in] matrix")
    if group_size not in _GROUPS:
        raise ValueError(f"group_size must be one of {_GROUPS}")
    if weight.numel() == 0:
        raise ValueError("weight must not be empty")
    dtype = weight.dtype if dtype is None else dtype
    out_dim, in_dim = weight.shape
    groups = -(-in_dim // group_size)
    w = weight.detach().float()
    pad = groups * group_size - in_dim
    if pad:  # the last group's absent columns repeat its last one: no change to its range
        w = torch.cat((w, w[:, -1:].expand(-1, pad)), dim=1)
    w = w.view(out_dim, groups, group_size)
    if zeros:
        low, high = w.amin(-1).clamp_max(0.0), w.amax(-1).clamp_min(0.0)
        scales = ((high - low) / 15.0).to(dtype)
        step = torch.where(scales == 0, torch.ones_like(scales), scales).float()
        zero = (-low / step).clamp_max(15.0).to(dtype)  # past 15 only by the rounding of the scale
        codes = torch.round(w / step[..., None] + zero.float()[..., None])
    else:
        scales = (w.abs().amax(-1) / 7.5).to(dtype)
        step = torch.where(scales == 0, torch.ones_like(scales), scales).float()
        zero = None
        codes = torch.round(w / step[..., None]) + 8.0
    codes = codes.clamp_(0, 15).to(torch.uint8).view(out_dim, -1)[:, :in_dim]
    if in_dim % 2:
        codes = F.pad(codes, (0, 1))
    return (codes[:, ::2] | codes[:, 1::2] << 4).contiguous(), scales.contiguous(), zero


def dequantize_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, in_dim: int, *,
                  group_size: int = 128) -> torch.Tensor:
    """The float32 ``[out, in_dim]`` weight that the codes stand for."""
    return _dequantize(codes, scales, zeros, in_dim, group_size, torch.float32)


def _dequantize(codes, scales, zeros, in_dim, group_size, dtype):
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1)[:, :in_dim].to(dtype)
    column = torch.arange(in_dim, device=codes.device) // group_size
    zero = 8.0 if zeros is None else zeros.to(dtype)[:, column]
    return (q - zero) * scales.to(dtype)[:, column]


def _validate(x, codes, scales, zeros, group_size) -> None:
    if group_size not in _GROUPS:
        raise ValueError(f"group_size must be one of {_GROUPS}")
    if x.dim() < 1 or codes.dim() != 2 or codes.dtype != torch.uint8:
        raise ValueError("codes must be a uint8 [out, ceil(in / 2)] matrix")
    in_dim, out_dim = x.shape[-1], codes.shape[0]
    if codes.shape[1] != (in_dim + 1) // 2:
        raise ValueError(f"expected {(in_dim + 1) // 2} bytes of codes a row for {in_dim} columns, got {codes.shape[1]}")
    want = (out_dim, -(-in_dim // group_size))
    if scales.shape != want or (zeros is not None and zeros.shape != want):
        raise ValueError(f"scales and zeros must have shape {want}")
    if zeros is not None and zeros.dtype != scales.dtype:
        raise ValueError("scales and zeros must have the same dtype")
    device = x.device
    if codes.device != device or scales.device != device or (zeros is not None and zeros.device != device):
        raise ValueError("linear_w4 tensors must be on the same device")


def linear_w4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
              group_size: int = 128) -> torch.Tensor:
    """``x [..., in] -> [..., out]`` with a 4-bit weight (see the module's description).

    On CUDA x is float16 or bfloat16, sums are float32 and the result is rounded once. Meant for
    decoding's few rows (up to 64 share one pass over the weight). Inference only: x must not require
    grad, on CUDA nor may scales and zeros.
    """
    _validate(x, codes, scales, zeros, group_size)
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("linear_w4 is inference only: x must not require grad")
    out_dim = codes.shape[0]
    if x.numel() == 0 or out_dim == 0:
        return x.new_zeros(*x.shape[:-1], out_dim)
    if not x.is_cuda:
        wide = torch.promote_types(x.dtype, torch.float32)
        return F.linear(x.to(wide), _dequantize(codes, scales, zeros, x.shape[-1], group_size, wide)).to(x.dtype)
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"linear_w4 needs float16 or bfloat16 activations on CUDA, got {x.dtype}")
    if torch.is_grad_enabled() and (scales.requires_grad or zeros is not None and zeros.requires_grad):
        raise ValueError("linear_w4 is inference only: scales and zeros must not require grad on CUDA")
    if _ext.has_tangent(x, scales, zeros):
        raise ValueError("linear_w4 is inference only: it has no forward-mode derivative on CUDA")
    if scales.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported scale dtype {scales.dtype}")
    if x.dim() == 2:
        return _ext.linear_w4(x, codes, scales, zeros, group_size)
    return _ext.linear_w4(x.reshape(-1, x.shape[-1]), codes, scales, zeros, group_size).view(*x.shape[:-1], out_dim)


class LinearW4(nn.Module):
    """An ``nn.Linear`` without bias on a 4-bit weight (buffers, so a ``state_dict`` carries it)."""

    def __init__(self, weight: torch.Tensor, *, group_size: int = 128, zeros: bool = False) -> None:
        super().__init__()
        codes, scales, zero = quantize_w4(weight, group_size=group_size, zeros=zeros)
        self.out_features, self.in_features = weight.shape
        self.group_size = group_size
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("zeros", zero)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.is_cuda and torch.is_autocast_enabled("cuda"):
            x = x.to(torch.get_autocast_dtype("cuda"))
        return linear_w4(x, self.codes, self.scales, self.zeros, group_size=self.group_size)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, group_size={self.group_size}"


def quantize_projections(model: nn.Module, *, group_size: int = 128, zeros: bool = False) -> nn.Module:
    """Replace every mixer's ``in_proj`` and ``out_proj`` in ``model`` by 4-bit ones, in place (a model
    that is refused stays as it was).

    The model is for inference from then on: run it under ``torch.no_grad()`` or ``inference_mode()``.
    In grad mode its ``forward`` raises, since a norm's weight requires grad and so do the projections'
    inputs. Scales and zero points take the weight's type."""
    found = [(module, name, layer) for module in model.modules() for name in ("in_proj", "out_proj")
             if isinstance(layer := getattr(module, name, None), nn.Linear)]
    for _, name, layer in found:
        if layer.bias is not None:
            raise ValueError(f"{name} has a bias: 4-bit projections have none")
    if group_size not in _GROUPS:
        raise ValueError(f"group_size must be one of {_GROUPS}")
    for module, name, layer in found:
        setattr(module, name, LinearW4(layer.weight, group_size=group_size, zeros=zeros))
    return model
