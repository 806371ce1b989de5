"""4-bit quantisation and its CPU product, and the orthogonalising optimiser off the GPU."""

from __future__ import annotations

import pytest
import torch

from _operator_refs import orthogonalize64, weight_w4
from mamba3_b200 import (GatedRecurrence, LinearW4, Mamba3, Muon, _ext, dequantize_w4, linear_w4, orthogonalize,
                         quantize_projections, quantize_w4)
from mamba3_b200.optim import COEFFICIENTS


@pytest.mark.parametrize("shape", [(5, 64), (3, 33), (7, 517), (2, 1)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_rounding_to_nearest(shape, group, zeros):
    w = torch.randn(shape, generator=torch.Generator().manual_seed(0))
    codes, scales, zero = quantize_w4(w, group_size=group, zeros=zeros)
    assert codes.dtype == torch.uint8 and codes.shape == (shape[0], (shape[1] + 1) // 2)
    back = dequantize_w4(codes, scales, zero, shape[1], group_size=group)
    torch.testing.assert_close(back.double(), weight_w4(codes, scales, zero, shape[1], group), rtol=1e-6, atol=1e-6)
    step = scales.repeat_interleave(group, 1)[:, :shape[1]]
    assert ((back - w).abs() <= 0.501 * step).all()


def test_groups_of_one_value():
    for value in (0.0, 0.3, -0.3):
        for zeros in (False, True):
            w = torch.full((2, 40), value)
            codes, scales, zero = quantize_w4(w, group_size=32, zeros=zeros)
            back = dequantize_w4(codes, scales, zero, 40, group_size=32)
            assert torch.isfinite(back).all()
            assert ((back - w).abs() <= 0.5001 * scales.amax()).all()


def test_product_and_shapes():
    w = torch.randn(19, 70)
    layer = LinearW4(w, group_size=32, zeros=True)
    x = torch.randn(2, 3, 70)
    y = layer(x)
    want = x.double() @ weight_w4(layer.codes, layer.scales, layer.zeros, 70, 32).t()
    torch.testing.assert_close(y.double(), want, rtol=1e-4, atol=1e-4)
    assert layer(torch.empty(0, 70)).shape == (0, 19)
    twin = LinearW4(torch.zeros(19, 70), group_size=32, zeros=True)
    twin.load_state_dict(layer.state_dict())
    assert torch.equal(twin(x), y)


def test_refusals():
    w = torch.randn(8, 64)
    codes, scales, _ = quantize_w4(w, group_size=64)
    x = torch.randn(2, 64)
    with pytest.raises(ValueError, match="group_size"):
        quantize_w4(w, group_size=48)
    with pytest.raises(ValueError, match="floating-point"):
        quantize_w4(codes)
    with pytest.raises(ValueError, match="must not be empty"):
        quantize_w4(torch.empty(0, 4))
    with pytest.raises(ValueError, match="group_size"):
        linear_w4(x, codes, scales, group_size=16)
    with pytest.raises(ValueError, match="bytes of codes"):
        linear_w4(x[:, :60], codes, scales, group_size=64)
    with pytest.raises(ValueError, match="must have shape"):
        linear_w4(x, codes, scales, group_size=32)
    with pytest.raises(ValueError, match="uint8"):
        linear_w4(x, codes.int(), scales, group_size=64)
    with pytest.raises(ValueError, match="same dtype"):
        linear_w4(x, codes, scales, scales.double(), group_size=64)
    with pytest.raises(ValueError, match="inference only"):
        linear_w4(x.requires_grad_(), codes, scales, group_size=64)
    with pytest.raises(ValueError, match="bias"):
        module = torch.nn.Module()
        module.in_proj = torch.nn.Linear(4, 4)
        quantize_projections(module)


@pytest.mark.parametrize("make", [lambda: Mamba3(64, d_state=16, depth=2), lambda: GatedRecurrence(64, depth=2),
                                  lambda: Mamba3(64, d_state=16, depth=1, causal=False)])
def test_quantised_models_stay_near(make):
    torch.manual_seed(0)
    model = make().eval()
    x = torch.randn(2, 20, 64)
    with torch.no_grad():
        want = model(x)
        quantize_projections(model, group_size=32)
        got = model(x)
        assert float((got - want).norm() / want.norm()) < 0.15
        if getattr(model, "causal", True):
            _, cache = model.prefill(x[:, :19])
            last, _ = model.step(x[:, 19:], cache)
            torch.testing.assert_close(last[:, 0], got[:, 19], rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("shape", [(1, 1), (5, 9), (9, 5), (2, 3, 12, 20)])
def test_orthogonalize_is_the_iterate_of_the_singular_values(shape):
    u = torch.randn(shape, generator=torch.Generator().manual_seed(0))
    got = orthogonalize(u, out_dtype=torch.float32)
    assert got.shape == u.shape
    torch.testing.assert_close(got.double(), orthogonalize64(u, 5, COEFFICIENTS), rtol=1e-3, atol=1e-4)
    assert (orthogonalize(torch.zeros(shape)) == 0).all()
    assert orthogonalize(torch.empty(0, 3)).shape == (0, 3)


def test_orthogonalize_refusals():
    with pytest.raises(ValueError, match="matrix"):
        orthogonalize(torch.randn(4))
    with pytest.raises(ValueError, match="steps"):
        orthogonalize(torch.randn(4, 4), steps=-1)
    with pytest.raises(ValueError, match="three numbers"):
        orthogonalize(torch.randn(4, 4), coefficients=(1.0, 2.0))


def test_muon_step_is_its_formula():
    torch.manual_seed(0)
    shapes = [(6, 4), (6, 4), (3, 8)]
    params = [torch.nn.Parameter(torch.randn(s)) for s in shapes]
    want = [p.detach().clone() for p in params]
    opt = Muon(params, lr=0.1, momentum=0.9, weight_decay=0.05)
    buffers = [torch.zeros(s) for s in shapes]
    for seed in range(3):
        for i, p in enumerate(params):
            p.grad = torch.randn(shapes[i], generator=torch.Generator().manual_seed(10 * seed + i))
            buffers[i] = 0.9 * buffers[i] + p.grad
            u = orthogonalize(p.grad + 0.9 * buffers[i]).float()
            want[i] = want[i] * (1 - 0.1 * 0.05) - 0.1 * max(1.0, shapes[i][0] / shapes[i][1]) ** 0.5 * u
        opt.step()
    for p, w in zip(params, want):
        torch.testing.assert_close(p.detach(), w, rtol=1e-5, atol=1e-5)


def test_muon_refusals():
    with pytest.raises(ValueError, match="matrices"):
        Muon([torch.nn.Parameter(torch.randn(3))])
    with pytest.raises(ValueError, match="momentum"):
        Muon([torch.nn.Parameter(torch.randn(3, 3))], momentum=1.0)


def test_packed_argument_structs_match_the_header():
    # int64 length + 4 ints + 14 tensors; 2 int64 + 4 ints + 5 tensors; 2 int64 + 3 ints + 3 floats + 3 tensors
    assert _ext._GATED_FORMAT.size == 24 + 14 * 64
    assert _ext._W4_FORMAT.size == 32 + 5 * 64
    assert _ext._ORTH_FORMAT.size == 40 + 3 * 64


def test_c_entries_reject_malformed_arguments_without_a_device():
    lib = _ext.load()
    absent = _ext._ABSENT
    for fn in (lib.m3_gated_scan_fwd, lib.m3_gated_scan_bwd, lib.m3_linear_w4, lib.m3_orthogonalize):
        assert fn(None, None) == 4
    assert lib.m3_gated_scan_fwd(_ext._GATED_FORMAT.pack(0, 1, 1, -1, 0, *absent * 14), None) == 1
    assert lib.m3_gated_scan_fwd(_ext._GATED_FORMAT.pack(4, 1, 1, -1, 0, *absent * 14), None) == 4
    assert b"value and forget" in lib.m3_last_error()
    assert lib.m3_linear_w4(_ext._W4_FORMAT.pack(4, 4, 1, 33, -1, 0, *absent * 5), None) == 1
    assert lib.m3_linear_w4(_ext._W4_FORMAT.pack(4, 4, 1, 32, -1, 0, *absent * 5), None) == 4
    assert lib.m3_orthogonalize(_ext._ORTH_FORMAT.pack(4, 4, 1, 65, -1, 1, 1, 1, *absent * 3), None) == 4
    assert lib.m3_orthogonalize(_ext._ORTH_FORMAT.pack(4, 4, 1, 5, -1, 1, 1, 1, *absent * 3), None) == 4
    assert lib.m3_orthogonalize_workspace_bytes(_ext._ORTH_FORMAT.pack(0, 4, 1, 5, -1, 1, 1, 1, *absent * 3)) == -1


def test_gated_entries_reject_widths_that_overflow():
    """Channels past the last block's are counted in 32 bits by the kernels: such widths end before a launch."""
    lib, absent = _ext.load(), _ext._ABSENT
    for length in (1, 4):
        for channels in (2 ** 31 - 1, 2 ** 31 - 4096):
            assert lib.m3_gated_scan_fwd(_ext._GATED_FORMAT.pack(length, 1, channels, -1, 0, *absent * 14), None) == 1
            assert lib.m3_gated_scan_bwd(_ext._GATED_FORMAT.pack(length, 1, channels, -1, 0, *absent * 14), None) == 1
    assert lib.m3_gated_scan_fwd(_ext._GATED_FORMAT.pack(1, 1, 2 ** 31 - 4097, -1, 0, *absent * 14), None) == 4


def test_muon_refuses_vectors_in_groups_added_later():
    p = torch.nn.Parameter(torch.randn(3, 4))
    opt = Muon([p])
    for vector in (torch.nn.Parameter(torch.randn(3)), torch.nn.Parameter(torch.tensor(1.0))):
        with pytest.raises(ValueError, match="matrices"):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.randn(2, 2)), vector]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": torch.nn.Parameter(torch.randn(2, 5)), "lr": 0.5})
    for group in opt.param_groups:
        for q in group["params"]:
            q.grad = torch.ones_like(q)
    opt.step()


@pytest.mark.parametrize("shape", [(0, 4), (4, 0)])
def test_muon_passes_empty_matrices_by(shape):
    empty, p = torch.nn.Parameter(torch.zeros(shape)), torch.nn.Parameter(torch.zeros(2, 3))
    opt = Muon([empty, p])
    empty.grad, p.grad = torch.zeros(shape), torch.ones(2, 3)
    opt.step()
    assert bool(p.abs().sum() > 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_muon_momentum_is_held_in_float32(dtype):
    """A momentum of 16 bits stands still once a gradient is below its last place: 0.95 m + g with m near 20 g."""
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(3, 4).to(dtype))
    opt, want = Muon([p], lr=0.0, momentum=0.99), torch.zeros(3, 4, dtype=torch.float64)
    for step in range(60):
        p.grad = (0.01 * torch.randn(3, 4, generator=torch.Generator().manual_seed(step)) + 0.1).to(dtype)
        want = 0.99 * want + p.grad.double()
        opt.step()
        if step == 30:  # through a checkpoint
            other = Muon([torch.nn.Parameter(p.detach().clone())], lr=0.0, momentum=0.99)
            other.load_state_dict(opt.state_dict())
            (p,), opt = other.param_groups[0]["params"], other
    held = opt.state[p]["momentum"]
    assert held.dtype == torch.float32 and p.dtype == dtype
    # 60 roundings of 2^-24 of at most the largest value, times 3 for the products
    assert float((held.double() - want).abs().max()) < 180 * 2.0 ** -24 * float(want.abs().max())


@pytest.mark.parametrize("zeros", [False, True])
def test_float64_products_off_the_gpu(zeros):
    w = torch.randn(9, 70, dtype=torch.float64)
    codes, scales, zero = quantize_w4(w, group_size=32, zeros=zeros)
    x = torch.randn(4, 70, dtype=torch.float64)
    want = x @ weight_w4(codes, scales, zero, 70, 32).t()
    torch.testing.assert_close(linear_w4(x, codes, scales, zero, group_size=32), want, rtol=1e-12, atol=1e-12)
    layer = LinearW4(w, group_size=32, zeros=zeros)
    torch.testing.assert_close(layer(x), want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_zero_points_lie_between_the_codes(dtype):
    """Negative weights alone put the zero point at 15, where the rounding of the scale must not carry it further: least of
    all a scale at the end of float16's range, which is half as large again or as small."""
    for size in (1.0, 0.8, 1.3e-6, 4e-7):
        w = -size * torch.rand(64, 32, generator=torch.Generator().manual_seed(0))
        codes, scales, zero = quantize_w4(w, group_size=32, zeros=True, dtype=dtype)
        assert float(zero.max()) <= 15.0 and float(zero.min()) >= 0.0
        back = dequantize_w4(codes, scales, zero, 32, group_size=32)
        # half a step, a step's unit of rounding over 15 codes and the zero point's own; clamped codes of a scale too small
        scale = scales.float()
        lost = (-w.amin(1, keepdim=True) - 15.0 * scale).clamp_min(0.0)
        assert bool(((back - w).abs() <= scale * (0.5 + 15 * 2.0 ** -8) + lost + (scale == 0) * size).all())


@pytest.mark.parametrize("group", [32, 48])
def test_a_refused_model_is_left_as_it_was(group):
    model = GatedRecurrence(64, depth=2)
    if group == 32:
        model.layers[1].mixer.out_proj = torch.nn.Linear(128, 64, bias=True)
    before = {name: type(module) for name, module in model.named_modules()}
    with pytest.raises(ValueError, match="bias|group_size"):
        quantize_projections(model, group_size=group)
    assert {name: type(module) for name, module in model.named_modules()} == before
