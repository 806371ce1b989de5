"""The gated-recurrence kernels against the token-by-token definition in 64 bits, forward and
gradients, over types, lengths around the tile, widths, strides, resets and extreme logits.

Bounds. A product f_t ... f_s and the sums are 32-bit: each step adds an error of at most about
4 units (2^-24) of the running state, random in sign; a state remembers at most min(L, 1 / (1 - f))
<= 1000 steps for the logits used here (f <= 0.999), so the sums are off by 4 * 2^-24 * sqrt(1000)
= 8e-6 of the largest state. Gradients are products of two such sums: twice that. On top comes one
rounding to the tensor's type."""

from __future__ import annotations

import threading

import pytest
import torch

from _operator_refs import assert_rounded, gated_scan64
from mamba3_b200 import GatedRecurrence, gated_scan, gated_step

pytestmark = pytest.mark.gpu
SUMS = 8e-6

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(batch, length, channels, dtype, gate=True, packed=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    parts = 3 if gate else 2
    projected = torch.randn(batch, length, parts * channels, device="cuda", generator=g)
    projected[..., channels:2 * channels] = projected[..., channels:2 * channels].mul(1.3).add(2.0).clamp(-6.0, 6.9)
    projected = projected.to(dtype)
    columns = [projected[..., i * channels:(i + 1) * channels] for i in range(parts)]
    if not packed:
        columns = [c.contiguous() for c in columns]
    state = torch.randn(batch, channels, device="cuda", generator=g)
    reset = torch.rand(batch, length, device="cuda", generator=g) < 0.05
    return columns[0], columns[1], columns[2] if gate else None, state, reset


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 300, 1025])
@pytest.mark.parametrize("channels", [1, 7, 64, 130])
def test_forward(dtype, length, channels):
    value, forget, gate, state, reset = _inputs(2, length, channels, dtype)
    for g, s, r in ((gate, state, reset), (None, None, None), (gate, None, None), (None, state, reset)):
        y, final = gated_scan(value, forget, g, initial_state=s, reset=r)
        want_y, want_final = gated_scan64(value, forget, g, s, r)
        assert y.dtype == dtype and final.dtype == torch.float32
        assert_rounded(y, want_y, SUMS, "y")
        assert_rounded(final, want_final, SUMS, "state")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("channels", [64, 129, 192])
def test_columns_of_a_projection_and_other_strides(dtype, channels):
    value, forget, gate, state, reset = _inputs(3, 150, channels, dtype, packed=True)
    want_y, want_final = gated_scan64(value, forget, gate, state, reset)
    y, final = gated_scan(value, forget, gate, initial_state=state, reset=reset)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)
    # time-major, channel-strided and broadcast inputs
    tm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    cs = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    y, final = gated_scan(tm(value), cs(forget), gate, initial_state=state.t().contiguous().t(),
                          reset=reset.t().contiguous().t())
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)
    shared = forget[:1].expand(3, -1, -1)
    y, final = gated_scan(value, shared, gate)
    want_y, want_final = gated_scan64(value, shared, gate)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)


@pytest.mark.parametrize("batch,length,channels", [(1, 9000, 64), (1, 5000, 130), (40, 200, 320), (2, 2100, 1024)])
def test_many_tiles(batch, length, channels):
    value, forget, gate, state, reset = _inputs(batch, length, channels, torch.bfloat16, packed=True)
    y, final = gated_scan(value, forget, gate, initial_state=state, reset=reset)
    want_y, want_final = gated_scan64(value, forget, gate, state, reset)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)


def _gradients(value, forget, gate, state, reset, dy, dstate, fn):
    leaves = [t.detach().requires_grad_() for t in (value, forget, gate, state) if t is not None]
    it = iter(leaves)
    v, f = next(it), next(it)
    g = next(it) if gate is not None else None
    s = next(it) if state is not None else None
    y, final = fn(v, f, g, s, reset)
    return torch.autograd.grad((y, final), leaves, (dy.to(y.dtype), dstate.to(final.dtype)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [1, 2, 64, 65, 300, 1025])
@pytest.mark.parametrize("channels", [7, 64, 130])
@pytest.mark.parametrize("gated", [True, False])
def test_backward(dtype, length, channels, gated):
    value, forget, gate, state, reset = _inputs(2, length, channels, dtype, gate=gated, packed=channels == 64)
    g = torch.Generator(device="cuda").manual_seed(5)
    dy = torch.randn(2, length, channels, device="cuda", generator=g).to(dtype)
    dstate = torch.randn(2, channels, device="cuda", generator=g)
    for s, r in ((state, reset), (None, None)):
        got = _gradients(value, forget, gate, s, r, dy, dstate,
                         lambda v, f, q, s_, r_: gated_scan(v, f, q, initial_state=s_, reset=r_))
        want = _gradients(value.double(), forget.double(), None if gate is None else gate.double(),
                          None if s is None else s.double(), r, dy, dstate, gated_scan64)
        for i, (a, e) in enumerate(zip(got, want)):
            assert_rounded(a, e, 2 * SUMS, f"gradient {i}")


def test_backward_many_tiles_and_strided_dy():
    value, forget, gate, state, reset = _inputs(2, 4200, 192, torch.float32, packed=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    dy = torch.randn(2, 192, 4200, device="cuda", generator=g).transpose(1, 2)
    dstate = torch.randn(2, 192, device="cuda", generator=g)
    got = _gradients(value, forget, gate, state, reset, dy, dstate,
                     lambda v, f, q, s, r: gated_scan(v, f, q, initial_state=s, reset=r))
    want = _gradients(value.double(), forget.double(), gate.double(), state.double(), reset, dy, dstate, gated_scan64)
    for a, e in zip(got, want):
        assert_rounded(a, e, 2 * SUMS)


@pytest.mark.parametrize("length", [650, 1300])
@pytest.mark.parametrize("channels", [128, 1216, 1300, 2368, 4736, 9600])
def test_every_split_of_a_sequence(length, channels):
    """1 to 16 CTAs walk a sequence's tiles together, by how many channels there are."""
    value, forget, gate, state, reset = _inputs(1, length, channels, torch.bfloat16, seed=channels)
    g = torch.Generator(device="cuda").manual_seed(6)
    dy = torch.randn(1, length, channels, device="cuda", generator=g).to(torch.bfloat16)
    dstate = torch.randn(1, channels, device="cuda", generator=g)
    run = lambda v, f, q, s, r: gated_scan(v, f, q, initial_state=s, reset=r)  # noqa: E731
    y, final = run(value, forget, gate, state, reset)
    want_y, want_final = gated_scan64(value, forget, gate, state, reset)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)
    got = _gradients(value, forget, gate, state, reset, dy, dstate, run)
    want = _gradients(value.double(), forget.double(), gate.double(), state.double(), reset, dy, dstate, gated_scan64)
    for i, (a, e) in enumerate(zip(got, want)):
        assert_rounded(a, e, 2 * SUMS, f"gradient {i}")


def test_gradient_against_differences():
    """The directional derivative of a float32 loss along a random direction, against a central difference
    of the 64-bit definition (error of the difference: about step^2 = 1e-8)."""
    value, forget, gate, state, reset = _inputs(2, 70, 33, torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(8)
    weight = torch.randn(2, 70, 33, device="cuda", generator=gen, dtype=torch.float64)
    leaves = [t.detach().requires_grad_() for t in (value, forget, gate, state)]
    y, final = gated_scan(leaves[0], leaves[1], leaves[2], initial_state=leaves[3], reset=reset)
    grads = torch.autograd.grad((y.double() * weight).sum() + final.double().sum(), leaves)
    ways = [torch.randn(t.shape, device="cuda", generator=gen, dtype=torch.float64) for t in leaves]
    slope = sum((g.double() * w).sum() for g, w in zip(grads, ways))

    def loss(step):
        moved = [t.detach().double() + step * w for t, w in zip(leaves, ways)]
        y64, f64 = gated_scan64(moved[0], moved[1], moved[2], moved[3], reset)
        return (y64 * weight).sum() + f64.sum()

    difference = (loss(1e-4) - loss(-1e-4)) / 2e-4
    assert abs(float(slope - difference)) < 1e-4 * max(1.0, float(sum(g.double().norm() * w.norm() for g, w in zip(grads, ways))) / 100)


def test_only_some_gradients():
    value, forget, gate, state, _ = _inputs(2, 100, 64, torch.bfloat16)
    forget.requires_grad_()
    y, final = gated_scan(value, forget, gate, initial_state=state)
    (grad,) = torch.autograd.grad(y.float().sum(), (forget,))  # the state's gradient is absent
    f64 = forget.detach().double().requires_grad_()
    y64, _ = gated_scan64(value, f64, gate, state)
    (want,) = torch.autograd.grad(y64.sum(), (f64,))
    assert_rounded(grad, want, 2 * SUMS)


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_logits(dtype):
    """Forget and gate logits at the ends of the type: f is 0 or 1 there, silu 0 or the gate."""
    value, forget, gate, state, _ = _inputs(1, 80, 66, dtype)
    forget[:, ::7] = -torch.inf
    forget[:, 3::7] = torch.inf
    forget[:, 5::7] = -1e4
    gate[:, ::5] = -1e4
    gate[:, 1::5] = 30.0
    y, final = gated_scan(value, forget, gate, initial_state=state)
    want_y, want_final = gated_scan64(value, forget, gate, state)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)


def test_nan_stays_in_its_channel_and_a_reset_ends_it():
    value, forget, gate, state, _ = _inputs(1, 200, 64, torch.float32)
    reset = torch.zeros(1, 200, dtype=torch.bool, device="cuda")
    reset[0, 150] = True
    value[0, 10, 3] = torch.nan
    forget[0, 20, 5] = torch.nan
    state[0, 9] = torch.inf
    y, final = gated_scan(value, forget, gate, initial_state=state, reset=reset)
    nan = torch.isnan(y)[0]
    assert nan[10:150, 3].all() and nan[20:150, 5].all()
    assert not nan[150:].any() and torch.isfinite(final).all()
    assert not nan[:, 4].any() and not torch.isfinite(y[0, 0, 9])


def test_reset_at_every_token():
    value, forget, gate, state, _ = _inputs(2, 130, 64, torch.float32)
    reset = torch.ones(2, 130, dtype=torch.bool, device="cuda")
    y, final = gated_scan(value, forget, gate, initial_state=state, reset=reset)
    want_y, want_final = gated_scan64(value, forget, gate, state, reset)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,channels", [(1, 5120), (3, 129), (64, 512), (257, 66)])
def test_step(dtype, batch, channels):
    value, forget, gate, state, _ = _inputs(batch, 1, channels, dtype, packed=True)
    for g in (gate, None):
        y, new = gated_step(value[:, 0], forget[:, 0], state, None if g is None else g[:, 0])
        want_y, want = gated_scan64(value, forget, g, state)
        assert y.shape == (batch, channels)
        assert_rounded(y, want_y[:, 0], SUMS)
        assert_rounded(new, want, SUMS)
        before = state.clone()
        y2, same = gated_step(value[:, 0], forget[:, 0], before, None if g is None else g[:, 0], out_state=before)
        assert same is before and torch.equal(before, new) and torch.equal(y2, y)


def test_step_under_a_cuda_graph():
    value, forget, gate, state, _ = _inputs(2, 1, 256, torch.bfloat16, packed=True)
    start = state.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        gated_step(value[:, 0], forget[:, 0], state, gate[:, 0], out_state=state)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = gated_step(value[:, 0], forget[:, 0], state, gate[:, 0], out_state=state)
    state.copy_(start)
    for _ in range(3):
        graph.replay()
    want = start
    for _ in range(3):
        want_y, want = gated_step(value[:, 0], forget[:, 0], want, gate[:, 0])
    assert torch.equal(state, want) and torch.equal(y, want_y)


def test_repeats_are_bitwise_equal_and_streams_are_respected():
    value, forget, gate, state, reset = _inputs(2, 3000, 320, torch.bfloat16, packed=True)
    first = gated_scan(value, forget, gate, initial_state=state, reset=reset)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = value * 1  # made on the side stream: the call has to run there, after it
        second = gated_scan(late, forget, gate, initial_state=state, reset=reset)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_refusals_on_cuda():
    value = torch.randn(2, 4, 3, device="cuda")
    with pytest.raises(TypeError, match="unsupported activation dtype"):
        gated_scan(value.double(), value.double())
    with pytest.raises(ValueError, match="state must be float32"):
        gated_scan(value, value, initial_state=torch.zeros(2, 3, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="same device"):
        gated_scan(value, value, initial_state=torch.zeros(2, 3))
    with pytest.raises(ValueError, match="does not support gradients"):
        gated_step(value[:, 0].requires_grad_(), value[:, 0], torch.zeros(2, 3, device="cuda"))


def test_module_on_the_gpu_matches_the_cpu():
    torch.manual_seed(0)
    model = GatedRecurrence(64, depth=2)
    x = torch.randn(2, 100, 64)
    want = model.double()(x.double())
    model = model.float().cuda()
    y = model(x.cuda())
    # float32 products of 64 and 128 terms through two blocks: about 1e-6 of the largest value
    assert_rounded(y.detach(), want.detach(), 1e-5)
    with torch.no_grad():
        out, cache = model.prefill(x[:, :99].cuda())
        last, _ = model.step(x[:, 99:].cuda(), cache)
        assert_rounded(last[:, 0], want[:, 99].detach(), 1e-5)
        again, _ = model.step(x[:, 99:].cuda(), cache, in_place=True)
        assert torch.equal(again, last)


def test_threads_with_different_shapes():
    """Calls of one kernel from several host threads, with clusters of 16 and of one CTA: the launches need
    different amounts of shared memory."""
    calls = [[t.contiguous() for t in torch.randn(3, 1, length, 64, device="cuda").bfloat16().unbind(0)]
             for length in (2048, 64)]
    want = [gated_scan(*x)[0] for x in calls]
    torch.cuda.synchronize()
    failed = []

    def work(x, expected):
        try:
            for _ in range(10000):
                y, _ = gated_scan(*x)
            if not torch.equal(y, expected):
                failed.append("another result")
        except RuntimeError as error:
            failed.append(str(error))

    threads = [threading.Thread(target=work, args=(calls[i % 2], want[i % 2])) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("length", [1, 3, 70])
@pytest.mark.parametrize("channels", [2, 8])
def test_more_sequences_than_a_grid_dimension(length, channels):
    """65,535 blocks go along a grid's y; the sequences past them and the last ones, which a rounded-up grid has too."""
    batch = 2 * 65535 + 5
    value, forget, gate, state, reset = _inputs(batch, length, channels, torch.bfloat16)
    y, final = gated_scan(value, forget, gate, initial_state=state, reset=reset)
    want_y, want_final = gated_scan64(value, forget, gate, state, reset)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)
    dy, dstate = torch.randn_like(value), torch.randn_like(state)
    got = _gradients(value, forget, gate, state, reset, dy, dstate,
                     lambda v, f, q, s, r: gated_scan(v, f, q, initial_state=s, reset=r))
    want = _gradients(value.double(), forget.double(), gate.double(), state.double(), reset, dy, dstate, gated_scan64)
    for a, e in zip(got, want):
        assert_rounded(a, e, 2 * SUMS)
    if length == 1:
        y, new = gated_step(value[:, 0], forget[:, 0], state, gate[:, 0])
        want_y, want = gated_scan64(value, forget, gate, state)
        assert_rounded(y, want_y[:, 0], SUMS)
        assert_rounded(new, want, SUMS)


@pytest.mark.parametrize("length", [650, 1300])
@pytest.mark.parametrize("channels", [128, 1216, 1300, 2368, 4736])
@pytest.mark.parametrize("gated", [True, False])
def test_every_split_of_a_float32_sequence(length, channels, gated):
    """Tiles of float32 leave room for fewer CTAs of a cluster, with a gate for fewer still."""
    value, forget, gate, state, reset = _inputs(1, length, channels, torch.float32, gate=gated, seed=channels)
    g = torch.Generator(device="cuda").manual_seed(6)
    dy = torch.randn(1, length, channels, device="cuda", generator=g)
    dstate = torch.randn(1, channels, device="cuda", generator=g)
    run = lambda v, f, q, s, r: gated_scan(v, f, q, initial_state=s, reset=r)  # noqa: E731
    y, final = run(value, forget, gate, state, reset)
    want_y, want_final = gated_scan64(value, forget, gate, state, reset)
    assert_rounded(y, want_y, SUMS)
    assert_rounded(final, want_final, SUMS)
    got = _gradients(value, forget, gate, state, reset, dy, dstate, run)
    want = _gradients(value.double(), forget.double(), None if gate is None else gate.double(), state.double(), reset, dy, dstate,
                      gated_scan64)
    for i, (a, e) in enumerate(zip(got, want)):
        assert_rounded(a, e, 2 * SUMS, f"gradient {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [1, 40, 700])
def test_masks_of_the_lowest_value(dtype, length):
    """Padding whose value is the type's lowest, before tokens whose forget logit drops the state: -inf, the lowest value,
    or -200, where float32's sigmoid is 0; and a state of that size from before. Nothing of it may be left."""
    lowest = torch.finfo(dtype).min
    for masked in (-torch.inf, lowest, -200.0):
        value, forget, gate, state, _ = _inputs(2, length, 70, dtype)
        first = torch.arange(length, device="cuda") % 23 == 0
        forget[:, first] = masked
        state[:] = torch.finfo(torch.float32).min
        value[:, torch.arange(length, device="cuda") % 23 == 22] = lowest
        y, final = gated_scan(value, forget, gate, initial_state=state)
        want_y, want_final = gated_scan64(value, forget, gate, state)
        padded = torch.arange(length, device="cuda") % 23 == 22
        assert_rounded(y[:, ~padded], want_y[:, ~padded], SUMS, "y")  # without the values that are as large as the mask
        if not padded[-1]:
            assert_rounded(final, want_final, SUMS, "state")
        if length == 1:
            y, new = gated_step(value[:, 0], forget[:, 0], state, gate[:, 0])
            assert_rounded(y, want_y[:, 0], SUMS)
            assert_rounded(new, want_final, SUMS)
        dy, dstate = torch.randn_like(value), torch.randn_like(state)
        got = _gradients(value, forget, gate, state, None, dy, dstate,
                         lambda v, f, q, s, r: gated_scan(v, f, q, initial_state=s, reset=r))
        want = _gradients(value.double(), forget.double(), gate.double(), state.double(), None, dy, dstate, gated_scan64)
        for name, a, e in zip(("value", "forget", "gate", "state"), got, want):
            if name == "value":
                assert_rounded(a, e, 2 * SUMS, name)
            elif name == "state":  # f is within 4 of float32's least numbers, 5.6e-45, and the gradients after it below 1e4
                assert float(a.abs().max()) <= 1e-40
