"""Rotary positions on the GPU against their definition in 64 bits (attn_ref.rotary)."""
import pytest
import torch

import attn_ref as R
import dihydrogen_b200 as dc
from test_gpu_ln import backend, tensor

pytestmark = pytest.mark.gpu

# n, heads, rotated heads, channels of a head, channels of (D,) H, W, dims
CASES = [
    (1, 1, 1, 2, (0, 2), (1, 1)),
    (2, 3, 2, 16, (8, 8), (5, 7)),
    (1, 6, 4, 32, (16, 16), (16, 16)),
    (1, 4, 4, 24, (8, 8, 8), (3, 4, 8)),
    (2, 5, 3, 48, (16, 16, 16), (5, 7, 9)),
    (1, 3, 2, 40, (12, 12, 14), (2, 3, 20)),   # channels of no axis
    (1, 9, 9, 64, (0, 30), (6, 10)),           # most channels of no axis
    (1, 2, 1, 7, (2, 4), (4, 6)),              # an odd head
    (1, 30, 20, 8, (2, 2, 4), (6, 10, 12)),
    (1, 2, 0, 8, (4, 4), (3, 5)),              # nothing is turned
    (1, 1, 1, 128, (40, 44, 44), (17, 33, 65)),
]
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("types", ["f32-f32", "f32-bf16", "bf16-bf16", "bf16-f32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(case, types, interleaved):
    n, heads, rotated, d, axis, dims = case
    a, b = (TYPES[t] for t in types.split("-"))
    g = torch.Generator().manual_seed(heads)
    x = torch.randn(n, heads * d, *dims, generator=g).to(a)
    be = backend()
    rot = dc.RotaryPositions(be, len(dims) + 2)
    tx, ty = tensor(x.cuda(), be), tensor(torch.empty(x.shape, dtype=b, device="cuda"), be)
    rot.setup(tx, d, list(reversed(axis)), rotated, base=100.0, interleaved=interleaved)
    for inverse, f in ((False, rot.forward), (True, rot.backward)):
        f(tx, ty)
        zero, one = [0] * len(dims), [1.0] * len(dims)
        R.close(ty.buffer, R.rotary(x, d, axis, rotated, 100.0, interleaved, zero, one, inverse, b), "turned")
    if a == b:  # in place, off alignment
        tz = tensor(x.cuda(), be, pad=1)
        rot.forward(tz, tz)
        rot.forward(tx, ty)
        assert torch.equal(tz.buffer, ty.buffer)


def test_far_positions_keep_their_angles():
    """A long row: the angles are worked out in 64 bits."""
    be = backend()
    x = torch.randn(1, 4, 1, 200003)
    rot = dc.RotaryPositions(be, 4)
    t, y = tensor(x.cuda(), be), tensor(x.cuda(), be)
    rot.setup(t, 4, [4, 0], step=[3.0, 1.0])
    rot.forward(t, y)
    R.close(y.buffer, R.rotary(x, 4, (0, 4), 1, 10000.0, False, [0, 0], [1.0, 3.0], False), "far")


def test_a_shard_has_the_angles_of_the_whole_tensor():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 24, 4, 9, 14, generator=g)
    want = R.rotary(x, 12, (4, 4, 4), 2, 100.0, False, [0] * 3, [1.0] * 3, False)
    for grid in ([2, 1, 1, 1, 1], [1, 2, 1, 1, 1], [1, 1, 2, 1, 1], [1, 1, 1, 1, 2]):
        for rank in range(2):
            be = backend()
            dist = dc.Distribution.make_overlapped_distribution(grid, [1 if s > 1 else 0 for s in grid])
            ts = [dc.Tensor([14, 9, 4, 24, 2], dc.Locale(rank, 2), dist) for _ in range(2)]
            for t in ts:
                t.allocate()
                t._storage.fill_(9.0)
            at = tuple(slice(o, o + l) for o, l in reversed(list(zip(ts[0].offset, ts[0].local_shape))))
            ts[0].owned().copy_(x[at])
            rot = dc.RotaryPositions(be, 5)
            rot.setup(ts[0], 12, [4, 4, 4], base=100.0)
            rot.forward(*ts)
            R.close(ts[1].owned(), (want[0][at], want[1][at]), "shard")
            ts[1].owned().fill_(9.0)
            assert bool((ts[1]._storage == 9.0).all())


def test_infinities_stay_where_nothing_is_turned():
    be = backend()
    x = torch.randn(1, 12, 2, 8)
    x[0, 6:] = float("inf")  # the second head is copied
    x[0, 4:6] = float("-inf")  # channels of no axis
    rot = dc.RotaryPositions(be, 4)
    t, y = tensor(x.cuda(), be), tensor(x.cuda(), be)
    rot.setup(t, 6, [2, 2], rotated_heads=1)
    rot.forward(t, y)
    assert torch.equal(y.buffer.cpu()[0, 4:], x[0, 4:]) and bool(torch.isfinite(y.buffer[0, :4]).all())


def test_captured():
    be = backend()
    x = torch.randn(1, 48, 12, 20)
    rot = dc.RotaryPositions(be, 4)
    t, y = tensor(x.cuda(), be), tensor(x.cuda().bfloat16(), be)
    rot.setup(t, 16, [8, 8])
    rot.forward(t, y)
    want = y.buffer.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rot.forward(t, y)
    y.buffer.zero_()
    graph.replay()
    assert torch.equal(y.buffer, want)
