"""The 4-bit projection kernel against the product in 64 bits, over types, rows, groups, ragged sizes,
strides and non-finite activations.

Bound. Code minus 8 and the 16-bit activations have exact products in float32; a row's sum of n
terms is off by at most n * 2^-24 of the sum of the terms' sizes (less in any other order of adding),
and each group's scale and zero point add a few units more: (n + 8) * 2^-24 * sum |x||w|, then one
rounding to the output's type."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from _operator_refs import TINY, UNIT, weight_w4
from mamba3_b200 import LinearW4, Mamba3, linear_w4, quantize_projections

pytestmark = pytest.mark.gpu


def _weight(out_dim, in_dim, group, zeros, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-in_dim // group)
    codes = torch.randint(0, 256, (out_dim, (in_dim + 1) // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(out_dim, groups, device="cuda", generator=g)) * 0.02).to(dtype)
    zero = (15.0 * torch.rand(out_dim, groups, device="cuda", generator=g)).to(dtype) if zeros else None
    return codes, scales, zero


def _check(x, codes, scales, zeros, group, y):
    rows = x.reshape(-1, x.shape[-1])
    w = weight_w4(codes, scales, zeros, x.shape[-1], group)
    want = rows.double() @ w.t()
    # |q x| + |z x|: the terms before they cancel
    size = rows.double().abs() @ (w.abs() + scales.double().abs().amax() * 16.0).t()
    got = y.reshape(want.shape).double()
    bound = UNIT[y.dtype] * want.abs() + (x.shape[-1] + 8) * 2.0 ** -24 * size + TINY[y.dtype]
    assert float(((got - want).abs() - bound).max()) <= 0.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 4, 7, 8, 9, 16, 33, 64, 65, 130])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows(dtype, rows, zeros):
    codes, scales, zero = _weight(300, 640, 64, zeros, dtype)
    x = torch.randn(rows, 640, device="cuda").to(dtype)
    y = linear_w4(x, codes, scales, zero, group_size=64)
    assert y.shape == (rows, 300) and y.dtype == dtype
    _check(x, codes, scales, zero, 64, y)


@pytest.mark.parametrize("out_dim,in_dim", [(1, 1), (1, 33), (16, 32), (37, 517), (130, 96), (64, 2048), (1000, 131), (24, 4098)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows", [1, 5, 20])
def test_sizes(out_dim, in_dim, group, zeros, rows):
    codes, scales, zero = _weight(out_dim, in_dim, group, zeros, torch.float16)
    x = torch.randn(rows, in_dim, device="cuda").to(torch.float16)
    _check(x, codes, scales, zero, group, linear_w4(x, codes, scales, zero, group_size=group))


@pytest.mark.parametrize("shape", [(10768, 2560), (2560, 5120)])
def test_model_sizes_and_float32_scales(shape):
    codes, scales, zero = _weight(*shape, 128, True, torch.float32)
    for rows in (1, 3, 64):
        x = torch.randn(rows, 1, shape[1], device="cuda").to(torch.bfloat16)
        y = linear_w4(x, codes, scales, zero)
        assert y.shape == (rows, 1, shape[0])
        _check(x, codes, scales, zero, 128, y)


def test_very_long_rows():
    """Thousands of groups with zero points, more than any table of them in shared memory would hold."""
    codes, scales, zero = _weight(20, 120000, 32, True, torch.float16)
    x = torch.randn(18, 120000, device="cuda").to(torch.float16)
    _check(x, codes, scales, zero, 32, linear_w4(x, codes, scales, zero, group_size=32))


def test_strides_and_offsets():
    codes, scales, zero = _weight(96, 256, 32, True, torch.bfloat16)
    wide = torch.randn(6, 515, device="cuda").to(torch.bfloat16)
    wide_codes = torch.zeros(96, 200, device="cuda", dtype=torch.uint8)
    wide_codes[:, 3:131] = codes
    for x in (wide[:, :256], wide[:, :256].repeat(5, 1), wide[:, 1:257].repeat(4, 1)[::2], wide[:, 1:257], wide[::2, 3:259], wide.t().contiguous().t()[:, :256], wide[:1].expand(6, -1)[:, :256]):
        for q in (codes, wide_codes[:, 3:131], codes.t().contiguous().t()):
            for s in (scales, scales.t().contiguous().t()):
                _check(x, q, s, zero, 32, linear_w4(x, q, s, zero, group_size=32))


@pytest.mark.parametrize("rows", [1, 8, 12, 40])
@pytest.mark.parametrize("in_dim,group", [(160, 32), (192, 64), (1120, 32), (2624, 64), (96, 32)])
def test_whole_groups_that_leave_a_short_end(rows, in_dim, group):
    codes, scales, zero = _weight(77, in_dim, group, rows % 8 == 0, torch.bfloat16)
    x = torch.randn(rows, in_dim, device="cuda").to(torch.bfloat16)
    _check(x, codes, scales, zero, group, linear_w4(x, codes, scales, zero, group_size=group))


@pytest.mark.parametrize("rows", [1, 3, 20, 64])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_unaligned_rows_between_other_values(rows, offset):
    """Rows of codes and of x that start anywhere, with NaN around x and other bytes around the codes."""
    out_dim, in_dim = 131, 1283
    codes, scales, zero = _weight(out_dim, in_dim, 32, offset % 2 == 1, torch.float16, seed=offset)
    scales, zero = scales.float(), None if zero is None else zero.float()
    bytes_ = codes.shape[1]
    flat = torch.full((offset + out_dim * bytes_,), 255, device="cuda", dtype=torch.uint8)
    packed = flat[offset:].view(out_dim, bytes_)
    packed.copy_(codes)
    wide = torch.full((rows, in_dim + 9), torch.nan, device="cuda", dtype=torch.float16)
    x = wide[:, offset:offset + in_dim]
    x.copy_(torch.randn(rows, in_dim, device="cuda"))
    _check(x, packed, scales, zero, 32, linear_w4(x, packed, scales, zero, group_size=32))


@pytest.mark.parametrize("rows", [5, 20, 40])
def test_rows_that_overlap(rows):
    """Windows over one signal: rows 8 columns apart."""
    codes, scales, zero = _weight(96, 256, 64, False, torch.bfloat16)
    x = torch.randn(8 * rows + 256, device="cuda").to(torch.bfloat16).as_strided((rows, 256), (8, 1))
    _check(x, codes, scales, zero, 64, linear_w4(x, codes, scales, zero, group_size=64))


def test_zero_scales_and_nonfinite_rows():
    codes, scales, zero = _weight(64, 256, 64, False, torch.bfloat16)
    scales[5] = 0.0
    x = torch.randn(4, 256, device="cuda").to(torch.bfloat16)
    x[2, 7] = torch.nan
    x[3, 100] = torch.inf
    y = linear_w4(x, codes, scales, zero, group_size=64)
    _check(x[:2], codes, scales, zero, 64, y[:2])
    assert torch.isnan(y[2]).all()
    w = weight_w4(codes, scales, zero, 256, 64)
    want = x[3].double() @ w.t()
    assert torch.equal(torch.isfinite(y[3]), torch.isfinite(want)) and (y[:2, 5] == 0).all()


def test_refusals_on_cuda():
    codes, scales, _ = _weight(16, 64, 64, False, torch.bfloat16)
    x = torch.randn(2, 64, device="cuda")
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        linear_w4(x, codes, scales, group_size=64)
    with pytest.raises(ValueError, match="same device"):
        linear_w4(x.bfloat16(), codes.cpu(), scales, group_size=64)
    with pytest.raises(ValueError, match="inference only"):
        linear_w4(x.bfloat16().requires_grad_(), codes, scales, group_size=64)


def test_another_stream_and_repeats():
    codes, scales, zero = _weight(2560, 5120, 128, True, torch.bfloat16)
    x = torch.randn(4, 5120, device="cuda").to(torch.bfloat16)
    first = linear_w4(x, codes, scales, zero)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = linear_w4(x * 1, codes, scales, zero)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)


@pytest.mark.parametrize("causal", [True, False])
def test_quantised_model_runs_the_dequantised_weights(causal):
    """Mamba3 with 4-bit projections against the same model whose weights are the dequantised ones."""
    torch.manual_seed(0)
    model = Mamba3(256, d_state=128, depth=2, causal=causal).cuda().to(torch.bfloat16).eval()
    twin = Mamba3(256, d_state=128, depth=2, causal=causal).cuda().to(torch.bfloat16).eval()
    twin.load_state_dict(model.state_dict())
    quantize_projections(model, group_size=64)
    for block, other in zip(model.layers, twin.layers):
        for name in ("in_proj", "out_proj"):
            q = getattr(block.mixer, name)
            assert isinstance(q, LinearW4)
            w = weight_w4(q.codes, q.scales, q.zeros, q.in_features, 64)
            getattr(other.mixer, name).weight.data.copy_(w)
    x = torch.randn(2, 40, 256, device="cuda", dtype=torch.bfloat16)
    with torch.inference_mode():
        want, got = twin(x), model(x)
        # bf16 weights round the dequantised ones (2^-9 each), two blocks of bf16 activations
        assert float((got.float() - want.float()).norm() / want.float().norm()) < 2e-2
        if causal:
            decoder = model.cuda_graph(batch_size=2)
            cache = None
            for t in range(4):
                y = decoder(x[:, t:t + 1])
                step, cache = model.step(x[:, t:t + 1], cache)
                assert float((y.float() - step.float()).norm() / step.float().norm()) < 1e-2
                assert float((step[:, 0].float() - want[:, t].float()).norm() / want[:, t].float().norm()) < 3e-2


def test_a_decoder_keeps_the_weights_that_its_graph_reads():
    """Projections are replaced, and the old ones dropped, after the capture."""
    torch.manual_seed(0)
    model = Mamba3(256, d_state=128, depth=2).cuda().to(torch.bfloat16).eval()
    quantize_projections(model, group_size=64)
    x = torch.randn(2, 1, 256, device="cuda", dtype=torch.bfloat16)
    decoder = model.cuda_graph(batch_size=2)
    read = [weakref.ref(t) for t in model.buffers()]
    want = decoder(x).clone()
    decoder.validate()
    for block in model.layers:
        for name in ("in_proj", "out_proj"):
            old = getattr(block.mixer, name)
            setattr(block.mixer, name, LinearW4(torch.randn(old.out_features, old.in_features, device="cuda").bfloat16(), group_size=64))
    del block, old
    gc.collect()
    assert all(ref() is not None for ref in read)  # and only then is the graph run again
    with pytest.raises(RuntimeError, match="recreate"):
        decoder.validate()
    decoder.reset()
    assert torch.equal(decoder(x), want)


def _check_nonfinite(x, codes, scales, zeros, group, y):
    """Infinities with their signs and NaN where the definition has them; finite outputs within the bound."""
    w = weight_w4(codes, scales, zeros, x.shape[-1], group)
    want = torch.stack([(row * w).sum(1) for row in x.double()])  # term by term: nothing but the definition's products
    bad = ~torch.isfinite(want)
    assert bool(bad.any())
    assert torch.equal(torch.nan_to_num(y.double()[bad], nan=0.5, posinf=1.0, neginf=-1.0),
                       torch.nan_to_num(want[bad], nan=0.5, posinf=1.0, neginf=-1.0))
    whole = torch.isfinite(x).all(1)
    if whole.any():
        _check(x[whole], codes, scales, zeros, group, y[whole])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 8, 9, 20, 64, 70])
@pytest.mark.parametrize("out_dim,in_dim,group", [(64, 256, 64), (300, 640, 128), (77, 517, 32), (130, 4160, 32)])
@pytest.mark.parametrize("zeros", [False, True])
def test_infinities_are_the_definitions(dtype, rows, out_dim, in_dim, group, zeros):
    codes, scales, zero = _weight(out_dim, in_dim, group, zeros, dtype)
    if zeros:
        zero = zero.round()  # zero points that some codes meet: infinity times 0 there
        zero[::3] = 8.0
    scales[1] = 0.0
    x = torch.randn(rows, in_dim, device="cuda").to(dtype)
    x[-1, in_dim // 2] = torch.inf
    if rows > 4:
        x[1, 3] = -torch.inf
        x[2, in_dim - 1] = torch.nan
        x[3, 0], x[3, in_dim - 1] = torch.inf, -torch.inf
    _check_nonfinite(x, codes, scales, zero, group, linear_w4(x, codes, scales, zero, group_size=group))


@pytest.mark.parametrize("rows", [2, 20, 64])
@pytest.mark.parametrize("zeros", [False, True])
def test_sums_that_only_the_scale_brings_back(rows, zeros):
    """Activations near the end of bfloat16's range: 7 times them is past float32's, a scale of 0.02 times that is not."""
    codes, scales, zero = _weight(300, 640, 64, zeros, torch.bfloat16)
    x = torch.randn(rows, 640, device="cuda").to(torch.bfloat16)
    x[1, 100] = 2e38
    y = linear_w4(x, codes, scales, zero, group_size=64)
    assert torch.isfinite(y).all()
    _check(x, codes, scales, zero, 64, y)


def test_scales_that_require_grad_are_refused():
    """The CPU form is differentiable in them; on CUDA the result would have no gradient, without a word."""
    codes, scales, zero = _weight(16, 64, 64, True, torch.bfloat16)
    x = torch.randn(2, 64, device="cuda").bfloat16()
    want = linear_w4(x, codes, scales, zero, group_size=64)
    for s, z in ((scales.clone().requires_grad_(), zero), (scales, zero.clone().requires_grad_())):
        with pytest.raises(ValueError, match="inference only"):
            linear_w4(x, codes, s, z, group_size=64)
        with torch.no_grad():
            assert torch.equal(linear_w4(x, codes, s, z, group_size=64), want)
