"""Newton-Schulz orthogonalisation on the GPU against the iterate of the singular values in 64 bits.

Bound. The operands of each product are 16-bit (unit 2^-11) with float32 sums. A rounding of X by 2^-11
of its Frobenius norm, spread over min(m, n) directions, is followed by at most five steps whose slope
is at most a = 3.4445 near 0 and below 1 at the fixed point; for matrices of a spectrum as here
(random, with strong directions of a few times its norm) the result is off by a few 1e-3 of its norm:
held to 4e-3, with a bfloat16 result's own rounding (2^-9, rms 1.7e-3) included."""

from __future__ import annotations

import pytest
import torch

from _operator_refs import orthogonalize64
from mamba3_b200 import GatedRecurrence, Muon, _ext, orthogonalize
from mamba3_b200.optim import COEFFICIENTS

pytestmark = pytest.mark.gpu
BOUND = 4e-3


def _update(count, rows, cols, dtype=torch.float32, seed=0, strong=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    rank = max(1, min(rows, cols) // 64)
    return (1e-3 * (make(count, rows, cols) + strong * make(count, rows, rank) @ make(count, rank, cols))).to(dtype)


def _off(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("shape", [(1, 1), (1, 200), (200, 1), (2, 3), (16, 16), (63, 65), (64, 64), (100, 37), (128, 256),
                                   (129, 130), (257, 255), (256, 1336), (1336, 256), (500, 700), (1000, 999)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_shapes(shape, dtype):
    u = _update(1, *shape, dtype)[0]
    got = orthogonalize(u)
    assert got.shape == shape and got.dtype == torch.bfloat16
    assert _off(got, orthogonalize64(u, 5, COEFFICIENTS)) < BOUND


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_stacks_and_output_types(out_dtype):
    u = _update(6, 96, 160).view(2, 3, 96, 160)
    got = orthogonalize(u, out_dtype=out_dtype)
    want = orthogonalize64(u, 5, COEFFICIENTS)
    assert got.dtype == out_dtype and got.shape == u.shape
    for i in range(2):
        for j in range(3):
            assert _off(got[i, j], want[i, j]) < BOUND


@pytest.mark.parametrize("steps", [0, 1, 2, 7])
@pytest.mark.parametrize("shape", [(80, 72), (72, 80)])
def test_steps_and_coefficients(steps, shape):
    u = _update(2, *shape)
    for co in (COEFFICIENTS, (2.0, -1.5, 0.5)):
        assert _off(orthogonalize(u, steps, coefficients=co), orthogonalize64(u, steps, co)) < BOUND


def test_scale_does_not_matter():
    u = _update(1, 130, 200)[0]
    want = orthogonalize64(u, 5, COEFFICIENTS)
    for scale in (1e-30, 1e-10, 1.0, 1e10, 1e30):
        assert _off(orthogonalize(u.double().mul(scale).float()), want) < BOUND


def test_strides():
    u = _update(2, 130, 200)
    want = orthogonalize64(u, 5, COEFFICIENTS)
    wide = torch.zeros(2, 130, 333, device="cuda")
    wide[:, :, 5:205] = u
    for v in (u.mT.contiguous().mT, wide[:, :, 5:205], u.permute(1, 0, 2).contiguous().permute(1, 0, 2)):
        assert _off(orthogonalize(v), want) < BOUND
    assert _off(orthogonalize(u[:1].expand(3, -1, -1))[2], want[0]) < BOUND


def test_zero_and_nonfinite_matrices_stay_apart():
    u = _update(4, 70, 90)
    u[1] = 0.0
    u[2, 3, 4] = torch.nan
    got = orthogonalize(u)
    want = orthogonalize64(u[[0, 3]], 5, COEFFICIENTS)
    assert _off(got[[0, 3]], want) < BOUND
    assert (got[1] == 0).all() and torch.isnan(got[2]).any()


def test_singular_values_come_near_one():
    got = orthogonalize(_update(1, 512, 1024)[0], out_dtype=torch.float32)
    s = torch.linalg.svdvals(got.double())
    assert float(s.max()) < 1.3 and float(s.min()) > 0.6


def test_streams_and_repeats():
    u = _update(2, 300, 520)
    first = orthogonalize(u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = orthogonalize(u * 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)


def test_refusals_on_cuda():
    with pytest.raises(TypeError, match="unsupported dtypes"):
        orthogonalize(torch.randn(3, 3, device="cuda", dtype=torch.float64))


def test_muon_steps_are_the_formula_and_lower_the_loss():
    """Each step moves a weight by lr * scale times the orthogonalised update: the 64-bit one, off by
    BOUND of its norm; over 10 steps on a layer stack the loss falls."""
    torch.manual_seed(0)
    model = GatedRecurrence(64, depth=2).cuda()
    matrices = [p for p in model.parameters() if p.dim() == 2]
    opt = Muon(matrices, lr=0.02, momentum=0.9, weight_decay=0.01)
    x = torch.randn(4, 130, 64, device="cuda")
    buffers = [torch.zeros_like(p) for p in matrices]
    losses = []
    for _ in range(10):
        loss = (model(x) - x.flip(-1)).square().mean()
        opt.zero_grad()
        loss.backward()
        before = [p.detach().clone() for p in matrices]
        buffers = [0.9 * m + p.grad for m, p in zip(buffers, matrices)]
        opt.step()
        losses.append(float(loss.detach()))
        for p, w, m in zip(matrices, before, buffers):
            scale = 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            moved = (w.double() * (1 - 0.02 * 0.01) - p.detach().double()) / scale
            assert _off(moved, orthogonalize64(p.grad + 0.9 * m, 5, COEFFICIENTS)) < BOUND
    assert losses[-1] < losses[0]


def _widths(count, rows, cols):
    args = _ext._ORTH_FORMAT.pack(rows, cols, count, 5, 0, 1.0, 1.0, 1.0, *_ext._ABSENT * 3)
    return tuple(_ext.load().m3_orthogonalize_tile(args, product) for product in range(3))


def _iterate64(u, steps, coefficients):
    """The definition in float64 products on the GPU, where the singular values take the CPU too long."""
    a, b, c = coefficients
    x = u.double()
    x = x.mT if u.shape[-2] > u.shape[-1] else x
    x = x / torch.linalg.matrix_norm(x, keepdim=True)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.mT if u.shape[-2] > u.shape[-1] else x


# stacks of matrices, and the tiles of X X^T, A A and P X on 148 SMs: pairs of CTAs (256), single ones with 128 or 64 columns.
# Only pairs ever have more tiles than places (74): 16 x 520 x 1030, 8 x 1030 x 1100 and the last three have.
TILES = [((1, 1100, 1300), (64, 64, 128)), ((4, 500, 700), (64, 64, 128)), ((4, 700, 900), (128, 128, 256)),
         ((5, 650, 660), (128, 128, 256)), ((1, 1030, 2100), (64, 64, 256)), ((1, 2100, 1030), (64, 64, 256)),
         ((2, 1270, 1280), (128, 128, 256)), ((16, 520, 1030), (256, 256, 256)), ((8, 1030, 1100), (256, 256, 256)),
         ((1, 2305, 2561), (256, 256, 256)), ((3, 2561, 1793), (256, 256, 256)), ((1, 3333, 3077), (256, 256, 256))]


@pytest.mark.parametrize("shape,widths", TILES)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_every_tile_of_the_products(shape, widths, out_dtype):
    assert _widths(*shape) == widths
    for dtype in (torch.float32, torch.bfloat16):
        u = _update(*shape, dtype, seed=shape[1])
        got = orthogonalize(u, out_dtype=out_dtype)
        want = _iterate64(u, 5, COEFFICIENTS)
        assert got.dtype == out_dtype
        for g, w in zip(got, want):
            assert _off(g, w) < BOUND
            # no element far from its own: an error of a tile or a triangle would be of the size of the entries
            assert float((g.double() - w).abs().max()) < 0.1 * float(w.abs().max())


@pytest.mark.parametrize("shape", [(8, 1030, 1100), (4, 700, 900), (1, 1100, 1300)])
def test_products_repeat_bitwise(shape):
    u = _update(*shape)
    first = orthogonalize(u, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(orthogonalize(u, out_dtype=torch.float32), first)
