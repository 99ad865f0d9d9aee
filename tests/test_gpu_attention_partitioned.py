"""The way of a spatially partitioned projection to the attention and back, on two emulated ranks: re-distributed to
sample-parallel in fp32, turned and rounded, attended to, and the gradient the same way back."""
import numpy as np
import pytest
import torch

import attn_ref as R
import dihydrogen_b200 as dc
import emu
from test_gpu_attention import heads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_partitioned_to_samples_and_back(dtype):
    n, h, d, dims = 2, 2, 16, (6, 10)
    shape = [dims[1], dims[0], 3 * h * d, n]
    g = np.random.default_rng(1).normal(size=tuple(reversed(shape))).astype(np.float32)
    dy = torch.randn(n, h * d, *dims, generator=torch.Generator().manual_seed(2)).to(dtype)
    locs = emu.locales(2)
    make = lambda grid, like=shape, t=torch.float32: [
        dc.Tensor(like, l, dc.Distribution.make_distribution(grid), dtype=t) for l in locs]
    cut, back, whole, dwhole = make([2, 1, 1, 1]), make([2, 1, 1, 1]), make([1, 1, 1, 2]), make([1, 1, 1, 2])
    small = shape[:2] + [h * d, n]
    r, dr = make([1, 1, 1, 2], t=dtype), make([1, 1, 1, 2], t=dtype)
    o, d_o = make([1, 1, 1, 2], small, dtype), make([1, 1, 1, 2], small, dtype)
    for t in cut:
        emu.scatter_owned(t, g)
    for ts in (back, whole, dwhole, r, dr, o, d_o):
        for t in ts:
            t.allocate()
    shufflers = [dc.TensorShuffler(a, b, connect=False) for a, b in zip(cut, whole)]
    for which in ("fwd", "bwd"):
        blobs = [s.export(which) for s in shufflers]
        for s in shufflers:
            s.connect(which, blobs)
    for s, t in zip(shufflers, cut):
        s.put("fwd", t.get_buffer())
    for s, t in zip(shufflers, whole):
        s.wait_unpack("fwd", t.get_buffer())
    be = dc.BackendDNNLib(dc.Locale(0, 1))
    lse = []
    for i in range(2):  # a sample each
        rot, at = dc.RotaryPositions(be, 4), dc.Attention(be, 4, h)
        rot.setup(whole[i], d, [8, 8], rotated_heads=2 * h)
        rot.forward(whole[i], r[i])
        parts, grads = ([t.channel_slice(j * h * d, h * d) for j in range(3)] for t in (r[i], dr[i]))
        lse.append(torch.empty(1, h, dims[0] * dims[1], device="cuda"))
        d_o[i].owned().copy_(dy[i:i + 1])
        at.forward(*parts, o[i], lse[i])
        at.backward(*parts, o[i], lse[i], d_o[i], *grads)
        rot.backward(dr[i], dwhole[i])
    for s, t in zip(shufflers, dwhole):
        s.put("bwd", t.get_buffer())
    for s, t in zip(shufflers, back):
        s.wait_unpack("bwd", t.get_buffer())
    torch.cuda.synchronize()
    assert all(s.status(w) == dc._abi.OK for s in shufflers for w in ("fwd", "bwd"))
    # every operator against its definition, of what it was given
    for i in range(2):
        turned = R.rotary(torch.from_numpy(g[i:i + 1]), d, (8, 8), 2 * h, 10000.0, False, [0, 0], [1.0, 1.0], False, dtype)
        R.close(r[i].buffer, turned, "turned")
        q, k, v = (heads(t, h) for t in r[i].buffer.cpu().split(h * d, 1))
        want = R.attention(q, k, v, d ** -0.5, d_o=heads(dy[i:i + 1], h), dtype=dtype)
        R.close(lse[i], want["lse"], "lse")
        R.close(heads(o[i].buffer, h), want["o"], "o")
        for name, t in zip(("dq", "dk", "dv"), dr[i].buffer.split(h * d, 1)):
            R.close(heads(t, h), want[name], name)
        turned_back = R.rotary(dr[i].buffer.cpu(), d, (8, 8), 2 * h, 10000.0, False, [0, 0], [1.0, 1.0], True)
        R.close(dwhole[i].buffer, turned_back, "gradient")
    got = emu.gather_owned(back, g.shape)
    assert np.array_equal(got, np.concatenate([t.buffer.cpu().numpy() for t in dwhole]))
