"""Elementwise gated linear recurrence: operators and a mixer stack built on them.

    f_t = sigmoid(forget_t);  h_t = f_t h_{t-1} + (1 - f_t) value_t;  y_t = h_t silu(gate_t)

per (batch, channel). :func:`gated_scan` runs whole sequences (differentiable), :func:`gated_step`
one token; :class:`GatedRecurrence` is a shape-preserving stack with ``forward``, ``prefill`` and
``step`` as ``Mamba3`` has them (``step`` can be captured in a CUDA graph).

Dispatch follows :mod:`mamba3_b200.ops`: CUDA tensors run the kernels of ``csrc/gated.cu`` (forward
and backward), with no other GPU path; CPU tensors run the PyTorch formulation below.
"""

from __future__ import annotations

import math

import torch
from torch import nn
from torch.nn import functional as F

from . import _ext
from .model import _project, _RMSNorm

_ACTIVATIONS = (torch.float32, torch.float16, torch.bfloat16)


def _validate(value, forget, gate, state, reset) -> None:
    if value.dim() != 3:
        raise ValueError("value must have shape [B, L, C]")
    shape = value.shape
    if forget.shape != shape or (gate is not None and gate.shape != shape):
        raise ValueError("forget and gate must match value's shape [B, L, C]")
    if forget.dtype != value.dtype or (gate is not None and gate.dtype != value.dtype):
        raise ValueError("value, forget and gate must have the same dtype")
    if state is not None and (state.dim() != 2 or state.shape[0] != shape[0] or state.shape[1] != shape[2]):
        raise ValueError(f"the state must have shape {(shape[0], shape[2])}")
    if reset is not None:
        if reset.shape != shape[:2]:
            raise ValueError(f"reset must have shape {tuple(shape[:2])}")
        if reset.dtype != torch.bool:
            raise ValueError("reset must be bool")
    device = value.device
    for t in (forget, gate, state, reset):
        if t is not None and t.device != device:
            raise ValueError("gated scan tensors must be on the same device")
    if value.is_cuda:
        if value.dtype not in _ACTIVATIONS:
            raise TypeError(f"unsupported activation dtype {value.dtype}")
        if state is not None and state.dtype != torch.float32:
            raise ValueError("the state must be float32")


def _places_differ(t: torch.Tensor) -> bool:
    """Whether the elements of a matrix lie in different places."""
    if t.is_contiguous():
        return True
    (rows, columns), (down, right) = t.shape, t.stride()
    if rows == 1 or columns == 1:
        return (down if columns == 1 else right) > 0
    common = math.gcd(down, right)
    # i down = j right first happens at i = right / common, j = down / common
    return down > 0 and right > 0 and (right // common >= rows or down // common >= columns)


def _elementwise_safe(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether a kernel that reads each element of ``t`` before it writes the same one of ``out``, in any order of
    elements, is right: they are one view, or they share no place (as far as the strides show it)."""
    if out is t:
        return True
    apart = out.data_ptr() - t.data_ptr()
    if out.dtype == t.dtype and out.stride() == t.stride():
        if apart == 0:
            return True
        (rows, columns), (down, right) = out.shape, out.stride()
        if right == 1 and down >= columns and apart % out.element_size() == 0:  # rows of one matrix, two parts of it perhaps
            i, j = divmod(apart // out.element_size(), down)
            return not (abs(i) < rows and j < columns or abs(i + 1) < rows and down - j < columns)

    def bytes_(m):
        return (sum((n - 1) * s for n, s in zip(m.shape, m.stride())) + 1) * m.element_size()

    return apart >= bytes_(t) or -apart >= bytes_(out)


def _scan_torch(value, forget, gate, state, reset):
    """Differentiable form in (at least) float32: neighbours at distances 1, 2, 4, ... joined."""
    wide = torch.promote_types(value.dtype, torch.float32)
    keep = torch.sigmoid(forget.to(wide))
    h = torch.sigmoid(-forget.to(wide)) * value.to(wide)
    if reset is not None:
        keep = keep.masked_fill(reset[..., None], 0.0)
    distance = 1
    while distance < value.shape[1]:
        h = torch.cat((h[:, :distance], h[:, distance:] + keep[:, distance:] * h[:, :-distance]), dim=1)
        keep = torch.cat((keep[:, :distance], keep[:, distance:] * keep[:, :-distance]), dim=1)
        distance *= 2
    if state is not None:
        h = h + keep * state.to(wide)[:, None]
    y = h if gate is None else h * F.silu(gate.to(wide))
    return y.to(value.dtype), h[:, -1]


class _GatedScan(torch.autograd.Function):
    """The recurrence on ``m3_gated_scan_fwd`` / ``m3_gated_scan_bwd``; the forward keeps the states
    before every tile of tokens, the backward recomputes the others from them."""

    @staticmethod
    def forward(ctx, value, forget, gate, state, reset):
        batch, length, channels = value.shape
        y = torch.empty(batch, length, channels, device=value.device, dtype=value.dtype)
        out = torch.empty(batch, channels, device=value.device, dtype=torch.float32)
        carry = _ext.gated_carry(value)
        _ext.gated_scan_forward(value, forget, gate, reset, state, y=y, out_state=out, carry=carry)
        ctx.save_for_backward(value, forget, gate, reset, carry)
        return y, out

    @staticmethod
    def backward(ctx, dy, dstate):
        if torch.is_grad_enabled():  # create_graph=True
            raise RuntimeError("gated_scan is differentiable once: its gradient has no gradient on CUDA")
        value, forget, gate, reset, carry = ctx.saved_tensors
        dy = torch.zeros(value.shape, device=value.device, dtype=value.dtype) if dy is None else dy
        dvalue, dforget, dgate, dinitial = _ext.gated_scan_backward(value, forget, gate, reset, carry, dy, dstate,
                                                                    want_initial=ctx.needs_input_grad[3])
        return dvalue, dforget, dgate, dinitial, None


def gated_scan(value: torch.Tensor, forget: torch.Tensor, gate: torch.Tensor | None = None, *,
               initial_state: torch.Tensor | None = None, reset: torch.Tensor | None = None):
    """The recurrence over whole sequences: ``(y [B, L, C], final state [B, C] float32)``.

    ``value``, ``forget`` (logits) and the optional output ``gate`` are ``[B, L, C]`` of one dtype
    (float32, float16 or bfloat16), of any strides: columns of one projection are read in place.
    On CUDA it has gradients in reverse mode, once; forward mode is refused.
    ``initial_state`` is ``[B, C]`` float32 (zeros without it). ``reset`` ``[B, L]`` (bool) marks
    tokens that start a document: they see a zero state, whatever it held. (A forget logit of -inf, or
    the type's lowest value, drops a finite state too.) The state is held in float32; ``y`` and the
    gradients are rounded once, to the inputs' dtype.
    """
    _validate(value, forget, gate, initial_state, reset)
    batch, length, channels = value.shape
    if value.numel() == 0:
        wide = torch.promote_types(value.dtype, torch.float32)
        state = (torch.zeros(batch, channels, device=value.device, dtype=wide) if initial_state is None
                 else initial_state.to(wide, copy=True))
        return value.clone(), state
    if not value.is_cuda:
        return _scan_torch(value, forget, gate, initial_state, reset)
    if _ext.has_tangent(value, forget, gate, initial_state):
        raise ValueError("gated_scan has no forward-mode derivative on CUDA")
    if torch.is_grad_enabled() and (value.requires_grad or forget.requires_grad
                                    or (gate is not None and gate.requires_grad)
                                    or (initial_state is not None and initial_state.requires_grad)):
        return _GatedScan.apply(value, forget, gate, initial_state, reset)
    y = torch.empty(batch, length, channels, device=value.device, dtype=value.dtype)
    state = torch.empty(batch, channels, device=value.device, dtype=torch.float32)
    _ext.gated_scan_forward(value, forget, gate, reset, initial_state, y=y, out_state=state)
    return y, state


def gated_step(value: torch.Tensor, forget: torch.Tensor, state: torch.Tensor, gate: torch.Tensor | None = None, *,
               out_state: torch.Tensor | None = None):
    """One token: ``(y [B, C], new state [B, C] float32)`` from ``value``, ``forget``, ``gate``
    ``[B, C]`` and the float32 ``state``. ``out_state`` receives the new state and may be ``state``
    itself (in-place decoding) or share memory with it in another way, but its elements lie in places of
    their own. Not differentiable on CUDA: sequences under autograd take :func:`gated_scan`."""
    if value.dim() != 2:
        raise ValueError("value must have shape [B, C]")
    if state is None:
        raise ValueError("gated_step needs a state; start from zeros")
    shape, dtype, device = value.shape, value.dtype, value.device
    if forget.shape != shape or state.shape != shape or (gate is not None and gate.shape != shape):
        raise ValueError("forget, gate and the state must match value's shape [B, C]")
    if forget.dtype != dtype or (gate is not None and gate.dtype != dtype):
        raise ValueError("value, forget and gate must have the same dtype")
    if forget.device != device or state.device != device or (gate is not None and gate.device != device):
        raise ValueError("gated step tensors must be on the same device")
    if out_state is not None and (out_state.shape != shape or out_state.dtype != torch.float32 or out_state.device != device):
        raise ValueError("out_state must be float32 and match the state's shape and device")
    if out_state is not None and not _places_differ(out_state):
        raise ValueError("out_state has several elements in one place")
    if not value.is_cuda or value.numel() == 0:
        if value.numel() == 0:
            y, new = value.clone(), state.clone()
        else:
            y, new = _scan_torch(value.unsqueeze(1), forget.unsqueeze(1), None if gate is None else gate.unsqueeze(1), state, None)
            y = y[:, 0]
        return y, new if out_state is None else out_state.copy_(new)
    if dtype not in _ACTIVATIONS:
        raise TypeError(f"unsupported activation dtype {dtype}")
    if state.dtype != torch.float32:
        raise ValueError("the state must be float32")
    if torch.is_grad_enabled() and (value.requires_grad or forget.requires_grad or state.requires_grad
                                    or (gate is not None and gate.requires_grad)):
        raise ValueError("gated_step does not support gradients on CUDA; use gated_scan")
    y = torch.empty(shape[0], shape[1], device=device, dtype=dtype)  # plain ints: half the time of a torch.Size
    if _ext.has_tangent(value, forget, gate, state):
        raise ValueError("gated_step has no forward-mode derivative on CUDA")
    new = out_state
    # threads take the elements in any order: what one still has to read must not be written by another
    if out_state is None or ((out_state is not state or dtype == torch.float32)
                             and not all(_elementwise_safe(out_state, t) for t in (state, value, forget, gate)
                                         if t is not None and t.dtype == torch.float32)):
        new = torch.empty(shape[0], shape[1], device=device, dtype=torch.float32)
    _ext.gated_step(value, forget, gate, state, y=y, out_state=new)
    return y, new if new is out_state or out_state is None else out_state.copy_(new)


class _GatedMixer(nn.Module):
    """in_proj -> gated recurrence -> out_proj."""

    def __init__(self, d_model: int) -> None:
        super().__init__()
        self.d_model = d_model
        self.d_inner = 2 * d_model
        self.in_proj = nn.Linear(d_model, 3 * self.d_inner, bias=False)
        # forget logits of time constants 2 to 1000 tokens, evenly spread over their logarithm
        spread = torch.exp(torch.linspace(math.log(2.0), math.log(1000.0), self.d_inner))
        self.forget_bias = nn.Parameter(torch.log(spread - 1.0))
        self.forget_bias._no_weight_decay = True
        self.out_proj = nn.Linear(self.d_inner, d_model, bias=False)

    def _columns(self, hidden: torch.Tensor):
        projected = _project(self.in_proj, hidden)
        value, forget, gate = projected.split(self.d_inner, dim=-1)
        return value, forget + self.forget_bias.to(projected.dtype), gate

    def forward(self, hidden, state=None, *, reset=None):
        value, forget, gate = self._columns(hidden)
        mixed, state = gated_scan(value, forget, gate, initial_state=state, reset=reset)
        return _project(self.out_proj, mixed), state

    def step(self, hidden, state, out_state=None):
        value, forget, gate = self._columns(hidden[:, 0])
        mixed, state = gated_step(value, forget, state, gate, out_state=out_state)
        return _project(self.out_proj, mixed).unsqueeze(1), state


class _GatedBlock(nn.Module):
    def __init__(self, d_model: int) -> None:
        super().__init__()
        self.norm = _RMSNorm(d_model)
        self.mixer = _GatedMixer(d_model)


class GatedRecurrence(nn.Module):
    """A shape-preserving stack of gated-recurrence mixers, ``[batch, length, d_model]`` in and out:
    RMSNorm -> mixer -> residual per block, RMSNorm at the end. It has no ``cuda_graph`` and no chunk
    sizes, and ``prefill`` starts from zero states.

    ``forward(x, reset=None)`` is differentiable; ``prefill(x)`` also returns the decode cache (one
    float32 ``[batch, 2 * d_model]`` state per layer); ``step(x, cache)`` processes one token, in place
    in the cache with ``in_place=True`` (on CUDA without gradients).
    """

    def __init__(self, d_model: int, depth: int = 4) -> None:
        super().__init__()
        if d_model <= 0:
            raise ValueError("d_model must be positive")
        if depth <= 0:
            raise ValueError("depth must be positive")
        self.d_model = d_model
        self.depth = depth
        self.layers = nn.ModuleList(_GatedBlock(d_model) for _ in range(depth))
        self.norm_f = _RMSNorm(d_model)
        with torch.no_grad():
            for layer in self.layers:
                layer.mixer.out_proj.weight.div_(math.sqrt(depth))

    def _validate_input(self, x: torch.Tensor, *, single_token: bool = False) -> None:
        if x.ndim != 3 or x.shape[-1] != self.d_model:
            raise ValueError(f"expected [batch, length, {self.d_model}], got {tuple(x.shape)}")
        if single_token and x.shape[1] != 1:
            raise ValueError(f"expected [batch, 1, {self.d_model}], got {tuple(x.shape)}")

    def _run(self, x, reset):
        states = []
        for layer in self.layers:
            mixed, state = layer.mixer(layer.norm(x), reset=reset)
            x = x + mixed
            states.append(state)
        return self.norm_f(x), states

    def forward(self, x: torch.Tensor, *, reset: torch.Tensor | None = None) -> torch.Tensor:
        self._validate_input(x)
        return self._run(x, reset)[0]

    def prefill(self, x: torch.Tensor, *, reset: torch.Tensor | None = None):
        """Process a prefix and return ``(output, cache)``."""
        self._validate_input(x)
        if x.shape[0] == 0 or x.shape[1] == 0:
            raise ValueError("prefill requires a non-empty batch and sequence")
        return self._run(x, reset)

    def allocate_cache(self, batch_size: int, *, device: torch.device) -> list[torch.Tensor]:
        return [torch.zeros(batch_size, 2 * self.d_model, device=device, dtype=torch.float32) for _ in self.layers]

    def step(self, x: torch.Tensor, cache=None, *, in_place: bool = False):
        """One token: ``(output [batch, 1, d_model], cache)``."""
        self._validate_input(x, single_token=True)
        if cache is None:
            cache = self.allocate_cache(x.shape[0], device=x.device)
        if len(cache) != len(self.layers):
            raise ValueError(f"expected cache for {len(self.layers)} layers")
        states = []
        for layer, state in zip(self.layers, cache):
            mixed, state = layer.mixer.step(layer.norm(x), state, out_state=state if in_place else None)
            x = x + mixed
            states.append(state)
        return self.norm_f(x), states
