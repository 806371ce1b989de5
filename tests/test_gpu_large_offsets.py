"""Tensors of more than 2^31 elements (10 to 30 GB on the device): what lies past the 32-bit offsets, against references of
the parts that are checked."""

from __future__ import annotations

import pytest
import torch

from _operator_refs import assert_rounded, gated_scan64, orthogonalize64, weight_w4
from mamba3_b200 import gated_scan, gated_step, linear_w4, orthogonalize
from mamba3_b200.optim import COEFFICIENTS

pytestmark = pytest.mark.gpu
SUMS = 8e-6  # as in the tests of the recurrence


@pytest.fixture(autouse=True)
def _memory():
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB of free device memory")
    yield
    torch.cuda.empty_cache()


def _random(*shape, dtype=torch.bfloat16, seed=0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("channels", [2048, 2055])  # columns that TMA reads, and that it does not
def test_a_long_sequence_and_its_gradients(channels):
    length = 2 ** 31 // channels + 5000
    value, forget, dy = (_random(1, length, channels, seed=i) for i in range(3))
    forget.add_(2.0).clamp_(-6.0, 6.75)
    reset = torch.zeros(1, length, dtype=torch.bool, device="cuda")
    starts = [700, length - 3000, length - 1000]
    reset[0, starts] = True  # documents: each is a sequence of its own
    leaves = [value.requires_grad_(), forget.requires_grad_()]
    y, final = gated_scan(value, forget, reset=reset)
    grads = torch.autograd.grad(y, leaves, dy)
    for first, last in ((0, 700), (length - 3000, length - 1000), (length - 1000, length)):
        part = slice(first, last)
        own = [t.detach()[:, part].double().requires_grad_() for t in (value, forget)]
        want_y, want_final = gated_scan64(*own)
        assert_rounded(y[:, part], want_y.detach(), SUMS)
        for got, want in zip(grads, torch.autograd.grad(want_y, own, dy[:, part].double())):
            assert_rounded(got[:, part], want, 2 * SUMS)
    assert_rounded(final, want_final.detach(), SUMS)


def test_many_decoded_sequences():
    batch, channels = 2 ** 31 // 8192 + 100, 8192
    value, forget = _random(batch, channels), _random(batch, channels, seed=1)
    state = _random(batch, channels, dtype=torch.float32, seed=2)
    tail = slice(batch - 200, batch)
    want_y, want = gated_scan64(value[tail, None], forget[tail, None], None, state[tail])
    y, new = gated_step(value, forget, state, out_state=state)
    assert_rounded(y[tail], want_y[:, 0], SUMS)
    assert_rounded(new[tail], want, SUMS)


@pytest.mark.parametrize("rows", [1, 8, 20, 64])
@pytest.mark.parametrize("bytes_", [32768, 32771])
def test_a_large_4_bit_weight(rows, bytes_):
    out_dim, in_dim, group = 2 ** 31 // bytes_ + 300, 2 * bytes_, 128
    generator = torch.Generator(device="cuda").manual_seed(0)
    codes = torch.randint(0, 256, (out_dim, bytes_), device="cuda", generator=generator, dtype=torch.uint8)
    scales = torch.rand(out_dim, -(-in_dim // group), device="cuda", generator=generator).mul_(0.02).bfloat16()
    x = _random(rows, in_dim, seed=3)
    y = linear_w4(x, codes, scales)
    for part in (slice(0, 64), slice(out_dim - 400, out_dim)):
        w = weight_w4(codes[part], scales[part], None, in_dim, group)
        want = x.double() @ w.t()
        size = x.double().abs() @ (w.abs() + 0.02 * 16.0).t()  # the bound of the products' own tests
        off = (y[:, part].double() - want).abs() - (2.0 ** -8 * want.abs() + (in_dim + 8) * 2.0 ** -24 * size)
        assert float(off.max()) <= 0.0


def test_a_large_stack():
    count, rows, cols = 2 ** 31 // (800 * 1000) + 50, 800, 1000
    update = _random(count, rows, cols)
    got = orthogonalize(update)
    for i in (0, count - 60, count - 1):
        want = orthogonalize64(update[i], 5, COEFFICIENTS)
        assert float((got[i].double().cpu() - want).norm() / want.norm()) < 4e-3  # as in the tests of its shapes
