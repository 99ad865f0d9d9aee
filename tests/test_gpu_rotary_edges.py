"""Rotary positions on the GPU: what a layer that was set up refuses, and what outlives it."""
import pytest
import torch

import attn_ref as R
import dihydrogen_b200 as dc
from test_gpu_ln import backend, tensor

pytestmark = pytest.mark.gpu


def shard(shape, grid, rank):
    t = dc.Tensor(shape, dc.Locale(rank, 2), dc.Distribution.make_distribution(grid))
    t.allocate()
    return t


def test_a_shard_at_another_place_is_refused():
    """Same local shape, other positions: the angles would be another shard's."""
    be = backend()
    shape = [12, 6, 8, 2]
    first, second, samples = shard(shape, [2, 1, 1, 1], 0), shard(shape, [2, 1, 1, 1], 1), shard(shape, [1, 1, 1, 2], 1)
    channels = shard([6, 6, 16, 2], [1, 1, 2, 1], 1)
    assert first.local_shape == second.local_shape == channels.local_shape
    rot = dc.RotaryPositions(be, 4)
    rot.setup(first, 4, [2, 2])
    rot.forward(first, first)
    for x, y in ((second, second), (first, second), (second, first), (channels, channels), (first, channels)):
        for f in (rot.forward, rot.backward):
            with pytest.raises(ValueError):
                f(x, y)
    rot.setup(samples, 4, [2, 2])  # other samples have the same positions
    rot.forward(samples, samples)
    half = shard(shape, [1, 1, 1, 2], 0)
    rot.forward(half, half)


def test_channel_slices_are_turned_in_place():
    """The queries of a packed projection alone, by a layer that is set up for a tensor like them."""
    be, g = backend(), torch.Generator().manual_seed(3)
    x = torch.randn(2, 20, 5, 8, generator=g)
    t = tensor(x.cuda(), be)
    part = t.channel_slice(4, 12)
    rot = dc.RotaryPositions(be, 4)
    rot.setup(tensor(torch.empty(2, 12, 5, 8, device="cuda"), be), 6, [2, 4])
    rot.forward(part, part)
    want = R.rotary(x[:, 4:16], 6, (4, 2), 2, 10000.0, False, [0, 0], [1.0, 1.0], False)
    R.close(t.buffer[:, 4:16], want, "turned")
    assert torch.equal(t.buffer[:, :4].cpu(), x[:, :4]) and torch.equal(t.buffer[:, 16:].cpu(), x[:, 16:])


def test_a_graph_outlives_another_setup():
    """The tables that a captured graph reads stay while the layer does; the same geometry again gets the same ones."""
    be = backend()
    x = torch.randn(1, 16, 12, 20)
    t, y = tensor(x.cuda(), be), tensor(torch.empty(x.shape, device="cuda"), be)
    other = tensor(torch.randn(1, 16, 40, 30).cuda(), be)
    rot = dc.RotaryPositions(be, 4)
    rot.setup(t, 16, [8, 8])
    rot.forward(t, y)
    want = y.buffer.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rot.forward(t, y)
    for base in (10.0, 100.0, 1000.0):
        rot.setup(other, 16, [4, 12], base=base)
        rot.forward(other, other)
    assert len(rot._plans) == 4
    rot.setup(t, 16, [8, 8])
    assert len(rot._plans) == 4
    y.buffer.zero_()
    graph.replay()
    assert torch.equal(y.buffer, want)
    y.buffer.zero_()
    rot.forward(t, y)
    assert torch.equal(y.buffer, want)


def test_tables_are_there_for_every_stream():
    """A kernel on a stream that waits for no other, straight behind the set-up."""
    s = torch.cuda.Stream()
    be = backend(s)
    x = torch.randn(1, 64, 1, 20001)
    t, y = tensor(x.cuda(), be), tensor(torch.empty(x.shape, device="cuda"), be)
    want = R.rotary(x, 64, (0, 64), 1, 10000.0, False, [0, 0], [1.0, 1.0], False)
    torch.cuda.synchronize()
    for _ in range(3):
        rot = dc.RotaryPositions(be, 4)
        rot.setup(t, 64, [64, 0])
        rot.forward(t, y)
        s.synchronize()
        R.close(y.buffer, want, "turned")
