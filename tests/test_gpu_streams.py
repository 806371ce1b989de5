"""The operators on a stream of the caller's whose inputs come late: behind a few milliseconds of other work, so that a
call which ran elsewhere, or before its inputs, would read what was there first."""

from __future__ import annotations

import pytest
import torch

from mamba3_b200 import gated_scan, gated_step, linear_w4, orthogonalize

pytestmark = pytest.mark.gpu


def _w4(rows, zeros):
    def make(g):
        codes = torch.randint(0, 256, (1000, 1280), device="cuda", generator=g, dtype=torch.uint8)
        scales, zero = (torch.rand(1000, 20, device="cuda", generator=g).bfloat16() for _ in range(2))
        return [torch.randn(rows, 2560, device="cuda", generator=g).bfloat16(), codes, scales] + [15 * zero] * zeros
    return make, linear_w4


def _scan(length):
    def make(g):
        return [torch.randn(2, length, 320, device="cuda", generator=g).bfloat16() for _ in range(3)] + [
            torch.randn(2, 320, device="cuda", generator=g)]
    return make, lambda v, f, q, s: gated_scan(v, f, q, initial_state=s)


def _training():
    make, _ = _scan(700)

    def run(*inputs):
        leaves = [t.detach().requires_grad_() for t in inputs]
        y, final = gated_scan(*leaves[:3], initial_state=leaves[3])
        return torch.autograd.grad((y, final), leaves, (inputs[0], inputs[3]))
    return make, run


def _step():
    def make(g):
        return [torch.randn(3, 512, device="cuda", generator=g).bfloat16() for _ in range(3)] + [
            torch.randn(3, 512, device="cuda", generator=g)]
    return make, lambda v, f, q, s: gated_step(v, f, s, q)


def _orth(*shape):
    return (lambda g: [torch.randn(*shape, device="cuda", generator=g)]), orthogonalize


CASES = {"w4 1 row": _w4(1, False), "w4 8 rows, zeros": _w4(8, True), "w4 16 rows": _w4(16, False), "w4 64 rows, zeros": _w4(64, True),
         "scan": _scan(3000), "scan of one token": _scan(1), "training": _training(), "step": _step(),
         "orthogonalize": _orth(2, 300, 520), "orthogonalize pairs": _orth(2, 1270, 1280)}


def _outputs(out):
    return [out] if isinstance(out, torch.Tensor) else list(out)


@pytest.mark.parametrize("name", list(CASES))
def test_inputs_that_come_late(name):
    make, run = CASES[name]
    inputs = [make(torch.Generator(device="cuda").manual_seed(seed)) for seed in range(3)]
    want = [_outputs(run(*x)) for x in inputs]
    assert not all(torch.equal(a, b) for a, b in zip(want[0], want[1]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    work = [torch.randn(8192, 8192, device="cuda").half() for _ in streams]
    held = [[t.clone() for t in inputs[2]] for _ in streams]  # other values
    torch.cuda.synchronize()
    for _ in range(3):
        got, late = [], []
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for _ in range(6):  # most of a millisecond each
                    torch.mm(work[i], work[i], out=work[i].clone())
                late.append(torch.cuda.Event())
                late[i].record()
                for to, t in zip(held[i], inputs[i]):
                    to.copy_(t)  # the kernel right before the call writes what it reads, weights too
                got.append(_outputs(run(*held[i])))
        ahead = not late[0].query()  # the calls were made while the first input was still to come
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
        for i in range(2):
            for to, t in zip(held[i], inputs[2]):
                to.copy_(t)
        torch.cuda.synchronize()
    assert ahead
