"""Calls of one kernel from several host threads, with sizes that need different amounts of shared memory."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

from mamba3_b200 import Mamba3, _ext

pytestmark = pytest.mark.gpu


def _run_together(calls, repeats):
    """Every call in two threads, `repeats` times; the errors."""
    failed = []

    def work(call):
        try:
            for _ in range(repeats):
                call()
        except RuntimeError as error:
            failed.append(str(error))

    threads = [threading.Thread(target=work, args=(call,)) for call in [*calls, *calls]]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return failed


def test_few_row_projections():
    lib, stream = _ext.load(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def call(columns):
        """m3_gemv with its struct filled once, so that most of a thread's time is in the entry point."""
        x, w = (torch.randn(rows, columns, device="cuda").bfloat16() for rows in (4, 8))
        y = torch.empty(4, 8, device="cuda", dtype=torch.bfloat16)
        args = _ext.GemvArgs(out_dim=8, in_dim=columns, rows=4, device=x.device.index)
        args.x, args.w, args.y = _ext._desc(x), _ext._desc(w), _ext._desc(y)

        def launch(keep=(x, w, y)):
            if lib.m3_gemv(ctypes.byref(args), stream):
                raise RuntimeError(lib.m3_last_error().decode())

        return launch

    assert not _run_together([call(16384), call(256)], 40000)


def _models():
    torch.manual_seed(0)
    return [(Mamba3(64, d_state=state, depth=1).cuda(), torch.randn(1, 70, 64, device="cuda")) for state in (128, 32)]


def test_float32_scans():
    def call(model, x):
        with torch.no_grad():
            model(x)

    assert not _run_together([lambda m=m, x=x: call(m, x) for m, x in _models()], 1500)


def test_training_kernels():
    def call(model, x):
        x = x.clone().requires_grad_()
        torch.autograd.grad(model(x).square().sum(), (x,))

    assert not _run_together([lambda m=m, x=x: call(m, x) for m, x in _models()], 300)
