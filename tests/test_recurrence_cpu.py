"""The gated recurrence off the GPU: its PyTorch form against the token-by-token definition, its
gradient against differences, the module's prefill / step agreement and every refusal."""

from __future__ import annotations

import pytest
import torch

from _operator_refs import gated_scan64
from mamba3_b200 import GatedRecurrence, _ext, gated_scan, gated_step, recurrence


def _inputs(batch, length, channels, dtype=torch.float64, gate=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64)  # noqa: E731
    value, forget = make(batch, length, channels), make(batch, length, channels) + 2.0
    return (value.to(dtype), forget.to(dtype), make(batch, length, channels).to(dtype) if gate else None,
            make(batch, channels))


@pytest.mark.parametrize("length", [1, 2, 3, 64, 129])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("with_reset", [True, False])
def test_torch_form_is_the_recurrence(length, gate, with_reset):
    value, forget, g, state = _inputs(2, length, 5, gate=gate)
    reset = torch.rand(2, length, generator=torch.Generator().manual_seed(1)) < 0.2 if with_reset else None
    y, final = gated_scan(value, forget, g, initial_state=state, reset=reset)
    want_y, want_final = gated_scan64(value, forget, g, state, reset)
    torch.testing.assert_close(y, want_y, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(final, want_final, rtol=1e-12, atol=1e-12)


def test_gradient_against_differences():
    value, forget, g, state = _inputs(2, 7, 3)
    reset = torch.zeros(2, 7, dtype=torch.bool)
    reset[0, 0] = reset[1, 4] = True
    leaves = [t.requires_grad_() for t in (value, forget, g, state)]
    assert torch.autograd.gradcheck(lambda v, f, q, s: gated_scan(v, f, q, initial_state=s, reset=reset), leaves)


def test_step_continues_a_scan():
    value, forget, g, state = _inputs(3, 9, 4)
    y, final = gated_scan(value, forget, g, initial_state=state)
    for t in range(9):
        out, state = gated_step(value[:, t], forget[:, t], state, g[:, t])
        torch.testing.assert_close(out, y[:, t], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(state, final, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("shape", [(0, 4, 3), (2, 0, 3), (2, 4, 0)])
def test_empty_inputs(shape):
    value = torch.empty(shape)
    state = torch.randn(shape[0], shape[2])
    y, final = gated_scan(value, value, value, initial_state=state)
    assert y.shape == shape
    torch.testing.assert_close(final, state)
    assert gated_scan(value, value)[1].shape == state.shape


def test_refusals():
    v = torch.randn(2, 4, 3)
    with pytest.raises(ValueError, match=r"\[B, L, C\]"):
        gated_scan(v[0], v[0])
    with pytest.raises(ValueError, match="match value's shape"):
        gated_scan(v, v[:, :3])
    with pytest.raises(ValueError, match="match value's shape"):
        gated_scan(v, v, v[:, :, :2])
    with pytest.raises(ValueError, match="same dtype"):
        gated_scan(v, v.double())
    with pytest.raises(ValueError, match="state must have shape"):
        gated_scan(v, v, initial_state=torch.zeros(3, 2))
    with pytest.raises(ValueError, match="reset must have shape"):
        gated_scan(v, v, reset=torch.zeros(2, 3, dtype=torch.bool))
    with pytest.raises(ValueError, match="reset must be bool"):
        gated_scan(v, v, reset=torch.zeros(2, 4))
    with pytest.raises(ValueError, match=r"\[B, C\]"):
        gated_step(v, v, torch.zeros(2, 3))
    with pytest.raises(ValueError, match="needs a state"):
        gated_step(v[:, 0], v[:, 0], None)
    with pytest.raises(ValueError, match="out_state must be float32"):
        gated_step(v[:, 0], v[:, 0], torch.zeros(2, 3), out_state=torch.zeros(2, 4))


def test_module_prefill_then_step_is_forward():
    torch.manual_seed(0)
    model = GatedRecurrence(32, depth=2).double().eval()
    x = torch.randn(2, 12, 32, dtype=torch.float64)
    with torch.no_grad():
        full = model(x)
        out, cache = model.prefill(x[:, :8])
        torch.testing.assert_close(out, full[:, :8], rtol=1e-9, atol=1e-9)
        for t in range(8, 12):
            out, cache = model.step(x[:, t:t + 1], cache)
            torch.testing.assert_close(out, full[:, t:t + 1], rtol=1e-9, atol=1e-9)


def test_module_refusals():
    with pytest.raises(ValueError, match="d_model"):
        GatedRecurrence(0)
    with pytest.raises(ValueError, match="depth"):
        GatedRecurrence(8, depth=0)
    model = GatedRecurrence(8, depth=1)
    with pytest.raises(ValueError, match="expected"):
        model(torch.randn(2, 3, 9))
    with pytest.raises(ValueError, match="non-empty"):
        model.prefill(torch.randn(2, 0, 8))
    with pytest.raises(ValueError, match=r"\[batch, 1, 8\]"):
        model.step(torch.randn(2, 2, 8))
    with pytest.raises(ValueError, match="cache for 1 layers"):
        model.step(torch.randn(2, 1, 8), [])


@pytest.mark.parametrize("shape", [(1, 1), (1, 4), (4, 1), (2, 3), (3, 2), (4, 5)])
def test_places_and_shared_memory_by_enumeration(shape):
    """Every pair of strides up to 6 and every distance up to 30 elements, against the sets of places."""
    buffer = torch.zeros(200)
    places = torch.arange(200)
    for down in range(7):
        for right in range(7):
            t = buffer.as_strided(shape, (down, right), 60)
            mine = places.as_strided(shape, (down, right), 60).flatten().tolist()
            assert recurrence._places_differ(t) == (len(set(mine)) == len(mine))
            for apart in range(-30, 31):
                other = places.as_strided(shape, (down, right), 60 + apart).flatten().tolist()
                safe = recurrence._elementwise_safe(buffer.as_strided(shape, (down, right), 60 + apart), t)
                shared = not set(other).isdisjoint(mine)
                assert not (safe and shared) or apart == 0
                if right == 1 and down >= shape[1]:  # rows of a matrix: never taken for shared when they are not
                    assert safe == (not shared) or apart == 0


def _out_states(state):
    """Destinations in the state's own memory: the state, shifted by an element and by a row, beside it, transposed."""
    rows, columns = state.shape
    for down, offset in ((columns, 0), (columns, 1), (columns, columns), (2 * columns, columns), (2 * columns, columns - 1)):
        buffer = torch.zeros((rows + 2) * 2 * columns, device=state.device)
        held = buffer.as_strided(state.shape, (down, 1))
        held.copy_(state)
        yield held, buffer.as_strided(state.shape, (down, 1), offset)
    square = state[:, :rows].contiguous()
    yield square, square.t()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_step_into_memory_shared_with_the_state(device):
    g = torch.Generator().manual_seed(0)
    value, forget, gate, state = (torch.randn(33, 600, generator=g).to(device) for _ in range(4))
    for held, out in _out_states(state):
        columns = held.shape[1]
        want_y, want = gated_step(value[:, :columns], forget[:, :columns], held.clone(), gate[:, :columns])
        y, new = gated_step(value[:, :columns], forget[:, :columns], held, gate[:, :columns], out_state=out)
        assert new is out and torch.equal(out, want) and torch.equal(y, want_y)
    # activations in the destination's memory
    buffer = torch.zeros(34, 600, device=device)
    buffer[1:] = value
    want_y, want = gated_step(value, forget, state)
    y, new = gated_step(buffer[1:], forget, state, out_state=buffer[:-1])
    assert torch.equal(new, want) and torch.equal(y, want_y)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_step_refuses_a_destination_of_shared_places(device):
    v, state = torch.randn(4, 6, device=device), torch.zeros(4, 6, device=device)
    buffer = torch.zeros(40, device=device)
    for out in (buffer[:6].expand(4, 6), buffer.as_strided((4, 6), (5, 1)), buffer.as_strided((4, 6), (1, 2))):
        with pytest.raises(ValueError, match="several elements"):
            gated_step(v, v, state, out_state=out)
        with pytest.raises(ValueError, match="several elements"):
            gated_step(v, v, out, out_state=out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("backward", [False, True])
def test_clusters_have_room(dtype, gate, backward):
    """Past 8 CTAs, which any GPU hosts, only where two of a cluster's CTAs fit an SM (227 KB, 1 KB of it a block's own,
    and 64 K registers) or, with a device to ask, where it hosts all clusters at once; and no more CTAs than there is
    room for on 148 SMs."""
    lib, size = _ext.load(), torch.empty((), dtype=dtype).element_size()
    threads, tensors, maps = (256, 4 if gate else 3, 16) if backward else (128, 3 if gate else 2, 4)
    sizes = set()
    for length in (2, 64, 129, 300, 640, 1024, 4096, 65536):
        for batch, channels in ((1, 64), (1, 128), (1, 640), (1, 1024), (2, 1000), (1, 1800), (3, 1001), (8, 2048), (70000, 3)):
            tensor = (1 << 20, _ext._TENSOR_CODES[dtype] | 3 << 32, 0, 0, 0, 0, 0, 0)
            args = _ext._GATED_FORMAT.pack(length, batch, channels, -1, 0, *tensor, *tensor, *(tensor if gate else _ext._ABSENT),
                                           *_ext._ABSENT * 11)
            cluster = lib.m3_gated_cluster(args, backward)
            memory = 2 * tensors * 64 * 64 * size + (maps + 2 * cluster) * 512 + 512 + 1024
            room = min(227 * 1024 // memory, 65536 // (128 * threads))
            assert cluster == 1 or cluster <= -(-length // 64)
            assert cluster <= 8 or room >= 2 or (torch.cuda.is_available() and cluster == 16)
            assert cluster == 1 or cluster * batch * -(-channels // 64) <= 148 * room
            sizes.add(cluster)
    assert sizes >= {1, 2, 4, 8}


@pytest.mark.parametrize("shape", [(2, 0, 3), (0, 4, 3), (2, 4, 0)])
def test_the_state_of_an_empty_sequence_is_a_tensor_of_its_own(shape):
    value, state = torch.empty(shape), torch.randn(shape[0], shape[2])
    _, final = gated_scan(value, value, initial_state=state)
    assert torch.equal(final, state)
    before = state.clone()
    final.add_(1.0)
    assert torch.equal(state, before)
