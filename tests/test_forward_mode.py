"""Forward-mode derivatives: the CPU forms carry tangents, the CUDA entry points refuse them (a kernel would
return a result without one, which reads as a derivative of zero)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mamba3_b200 import GatedRecurrence, LinearW4, gated_scan, gated_step, linear_w4, orthogonalize, quantize_w4
from mamba3_b200.model import _project


def _operands(device, dtype):
    g = torch.Generator().manual_seed(0)
    make = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64).to(device, dtype)  # noqa: E731
    codes, scales, zeros = quantize_w4(make(24, 64), group_size=32, zeros=True)
    return {
        "scan": (lambda v, f, q, s: gated_scan(v, f, q, initial_state=s)[0],
                 [make(2, 9, 8), make(2, 9, 8), make(2, 9, 8), make(2, 8)]),
        "scan without gate": (lambda v, f: gated_scan(v, f)[1], [make(2, 9, 8), make(2, 9, 8)]),
        "step": (lambda v, f, s, q: gated_step(v, f, s, q)[0], [make(2, 8) for _ in range(4)]),
        "w4": (lambda x, s, z: linear_w4(x, codes, s, z, group_size=32), [make(3, 64), scales, zeros]),
        "orthogonalize": (lambda u: orthogonalize(u, out_dtype=torch.float32), [make(12, 20)]),
    }


NAMES = list(_operands("cpu", torch.float32))


@pytest.mark.parametrize("name", NAMES)
def test_the_cpu_forms_carry_tangents(name):
    fn, operands = _operands("cpu", torch.float32)[name]
    for i, t in enumerate(operands):
        along = torch.randn_like(t)
        with forward_ad.dual_level():
            out = forward_ad.unpack_dual(fn(*operands[:i], forward_ad.make_dual(t, along), *operands[i + 1:])).tangent
        step = 1e-3
        ends = [fn(*operands[:i], t + s * along, *operands[i + 1:]) for s in (step, -step)]
        torch.testing.assert_close(out, (ends[0] - ends[1]) / (2 * step), rtol=0.02, atol=0.02)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_cuda_refuses_tangents(name, grad):
    dtype = torch.bfloat16 if name == "w4" else torch.float32
    fn, operands = _operands("cuda", dtype)[name]
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        fn(*operands)  # tensors without a tangent go as ever
        for i, t in enumerate(operands):
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                fn(*operands[:i], forward_ad.make_dual(t, torch.ones_like(t)), *operands[i + 1:])
    with pytest.raises(Exception, match="forward-mode|data pointer"):
        torch.func.jvp(lambda t: fn(t, *operands[1:]), (operands[0],), (torch.ones_like(operands[0]),))


@pytest.mark.gpu
def test_few_row_projections_keep_tangents():
    layer = torch.nn.Linear(256, 64, bias=False).cuda().bfloat16()
    x, along = torch.randn(2, 2, 256, device="cuda").bfloat16().unbind(0)
    with torch.no_grad(), forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(_project(layer, forward_ad.make_dual(x, along))).tangent
        assert torch.equal(tangent, torch.nn.functional.linear(along, layer.weight))


@pytest.mark.gpu
def test_modules_refuse_tangents():
    model = GatedRecurrence(64, depth=1).cuda()
    layer = LinearW4(torch.randn(16, 64, device="cuda").bfloat16())
    for call, dtype in ((model, torch.float32), (model.step, torch.float32), (layer, torch.bfloat16)):
        x = torch.randn(2, 1, 64, device="cuda").to(dtype)
        with torch.no_grad(), forward_ad.dual_level():
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
