"""Layouts that the operators of attention between cells refuse because a rank would work out something else than the
whole tensor's result: no GPU."""
import pytest
import torch

import dihydrogen_b200 as dc


class Backend:
    stream = None


def shard(shape, grid, rank=0, dtype=torch.float32):
    size = 1
    for e in grid:
        size *= e
    t = dc.Tensor(shape, dc.Locale(rank, size), dc.Distribution.make_distribution(grid), dtype=dtype)
    t.allocate("cpu")
    return t


def test_layer_norm_needs_all_channels_of_a_cell():
    ln = dc.LayerNormalization(Backend(), 4, 1e-5)
    x, whole = shard([6, 4, 8, 2], [1, 1, 2, 1]), shard([6, 4, 4, 2], [1, 1, 1, 1])
    assert x.local_shape == whole.local_shape
    for a, b in ((x, x), (whole, x), (x, whole)):
        with pytest.raises(ValueError, match="channels of a cell"):
            ln.forward(a, None, None, b)
    for args in ((x, whole, whole), (whole, x, whole), (whole, whole, x)):
        with pytest.raises(ValueError, match="channels of a cell"):
            ln.backward(*args[:2], None, None, None, None, None, args[2])


def test_rotary_positions_need_all_channels_of_a_cell():
    rot = dc.RotaryPositions(Backend(), 4)
    with pytest.raises(ValueError, match="channels of a cell"):
        rot.setup(shard([6, 4, 8, 2], [1, 1, 2, 1]), 4, [2, 2])


def test_channel_slices_lie_where_their_tensor_does():
    t = shard([6, 4, 8, 2], [2, 1, 1, 1], rank=1)
    assert t.offset == [3, 0, 0, 0] and t.channel_slice(5, 2).offset == [3, 0, 5, 0]


def test_redistribution_of_16_bits_is_refused_with_the_way_round():
    a, b = shard([6, 4, 8, 2], [2, 1, 1, 1], dtype=torch.bfloat16), shard([6, 4, 8, 2], [1, 1, 1, 2], dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="before the rounding"):
        dc.TensorShuffler(a, b, connect=False)
    part = shard([6, 4, 8, 2], [2, 1, 1, 1])
    with pytest.raises(ValueError, match="in torch.float32"):
        dc.Attention(Backend(), 4, 2).forward(part, part, part, part, None)


def test_rotary_positions_without_a_setup():
    rot, x = dc.RotaryPositions(Backend(), 4), shard([6, 4, 8, 2], [1, 1, 1, 1])
    with pytest.raises(ValueError, match="setup"):
        rot.forward(x, x)
    with pytest.raises(dc._abi.DcbError):
        rot.setup(x, 4, [3, 1])  # axes have pairs of channels
    with pytest.raises(ValueError, match="setup"):
        rot.backward(x, x)
