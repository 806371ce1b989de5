"""64-bit references of the recurrence, 4-bit projection and orthogonalisation, and the rounding
bounds that the GPU tests hold the kernels to."""

from __future__ import annotations

import torch

# unit roundoffs 2^-p of significands of p = 24, 11 and 8 bits: one rounding of v is off by at most UNIT * |v|
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# smallest normal step of a type: below it a rounding is off by up to half of this, whatever the value
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def assert_rounded(actual, expected, sums: float, name: str = "") -> None:
    """``actual`` is ``expected`` (64 bits) up to one rounding to its type and ``sums`` times the
    largest expected value (the error of the 32-bit arithmetic before it)."""
    assert torch.equal(torch.isnan(actual).cpu(), torch.isnan(expected).cpu()), name
    e = torch.nan_to_num(expected.double().cpu())
    a = torch.nan_to_num(actual.double().cpu())
    largest = float(e.abs().max()) if e.numel() else 0.0
    unit = UNIT[actual.dtype]
    allowed = unit * e.abs() + (1.0 + unit) * sums * largest + TINY[actual.dtype]
    worst = float(((a - e).abs() - allowed).max()) if e.numel() else -1.0
    assert worst <= 0.0, f"{name}: {worst:.3g} over the bound (largest value {largest:.3g})"


def gated_scan64(value, forget, gate=None, state=None, reset=None):
    """The recurrence token by token in float64, differentiable."""
    value, forget = value.double(), forget.double()
    batch, length, channels = value.shape
    h = value.new_zeros(batch, channels) if state is None else state.double()
    keep, lose = torch.sigmoid(forget), torch.sigmoid(-forget)
    hs = []
    for t in range(length):
        if reset is not None:
            h = torch.where(reset[:, t, None], torch.zeros_like(h), h)
        h = keep[:, t] * h + lose[:, t] * value[:, t]
        hs.append(h)
    y = torch.stack(hs, 1)
    if gate is not None:
        g = gate.double()
        y = y * g * torch.sigmoid(g)
    return y, h


def weight_w4(codes, scales, zeros, in_dim, group):
    """The float64 weight that 4-bit codes stand for."""
    out_dim = codes.shape[0]
    w = torch.empty(out_dim, in_dim, dtype=torch.float64, device=codes.device)
    w[:, ::2] = (codes & 15).double()[:, :(in_dim + 1) // 2]
    w[:, 1::2] = (codes >> 4).double()[:, :in_dim // 2]
    for g in range(-(-in_dim // group)):
        cols = slice(g * group, min(in_dim, (g + 1) * group))
        zero = 8.0 if zeros is None else zeros[:, g:g + 1].double()
        w[:, cols] = (w[:, cols] - zero) * scales[:, g:g + 1].double()
    return w


def orthogonalize64(update, steps, coefficients):
    """The iterate through the singular values: each step maps s to a s + b s^3 + c s^5."""
    a, b, c = coefficients
    u, s, vt = torch.linalg.svd(update.double().cpu(), full_matrices=False)
    norm = s.square().sum(-1, keepdim=True).sqrt()
    s = s / torch.where(norm == 0, torch.ones_like(norm), norm)
    for _ in range(steps):
        s = s * (a + s * s * (b + c * s * s))
    return (u * s[..., None, :]) @ vt
