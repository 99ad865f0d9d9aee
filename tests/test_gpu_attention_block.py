"""A block of a network - layer norm, a 1 x 1 convolution, rotary positions, attention, and all their gradients - captured
into a graph and replayed with other inputs, against the same calls by themselves."""
import pytest
import torch

import dihydrogen_b200 as dc
from test_gpu_ln import backend, tensor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
def test_a_captured_block(masked, dtype):
    be, g = backend(), torch.Generator(device="cuda").manual_seed(1)
    n, c, h, d, dims = 2, 16, 2, 16, (12, 20)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    new = lambda ch, t=torch.float32: tensor(torch.zeros(n, ch, *dims, dtype=t, device="cuda"), be)
    x, u, du, dx, qkv, dqkv = (new(ch) for ch in (c, c, c, c, 3 * h * d, 3 * h * d))
    r, dr, o, d_o = (new(ch, dtype) for ch in (3 * h * d, 3 * h * d, h * d, h * d))
    w, gamma, beta = rnd(3 * h * d, c, 1, 1) / 4, rnd(c), rnd(c)
    dw, dg, db = torch.zeros_like(w), torch.zeros_like(gamma), torch.zeros_like(beta)
    ln, rot, at, conv = dc.LayerNormalization(be, 4, 1e-5), dc.RotaryPositions(be, 4), dc.Attention(be, 4, h), dc.Convolution(be, 4)
    conv.setup(u, w, qkv, du, dw, dqkv, [0, 0], [1, 1], [1, 1])
    rot.setup(qkv, d, [8, 8], rotated_heads=2 * h)
    mean, inv = ln.new_statistics(x)
    lse = torch.zeros(n, h, dims[0] * dims[1], device="cuda")
    mask = torch.ones(n, dims[0] * dims[1], dtype=torch.bool, device="cuda") if masked else None
    cut = lambda t: [t.channel_slice(i * h * d, h * d) for i in range(3)]

    def step():
        ln.forward(x, gamma, beta, u, mean, inv)
        conv.forward(1.0, u, w, 0.0, qkv)
        rot.forward(qkv, r)
        at.forward(*cut(r), o, lse, q_mask=mask, kv_mask=mask)
        at.backward(*cut(r), o, lse, d_o, *cut(dr), q_mask=mask, kv_mask=mask)
        rot.backward(dr, dqkv)
        conv.backward_data(1.0, w, dqkv, 0.0, du)
        conv.backward_filter(1.0, u, dqkv, 0.0, dw)
        ln.backward(x, du, mean, inv, gamma, dg, db, dx)

    same = [t.buffer for t in (u, qkv, r, o, dr, dqkv)] + [lse, mean, inv]
    # backward data adds its parts up in the order in which they are done: what follows it agrees up to roundings of sums
    # of 96 products and, behind them, of 16 channels and 480 cells
    near = [du.buffer, dx.buffer, dw, dg, db]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(5):
        x.buffer.copy_(rnd(n, c, *dims))
        d_o.buffer.copy_(rnd(n, h * d, *dims))
        if masked:
            mask.copy_(rnd(*mask.shape) < 0.7)
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in same], [t.clone() for t in near]
        for t in same + near:
            t.fill_(float("nan"))
        for _ in range(3):  # one replay straight behind the other
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(same, want[0]):
            assert torch.equal(a, b)
        for a, b in zip(near, want[1]):
            assert float((a - b).abs().max()) <= (96 + 16 + 480) * 2.0 ** -24 * float(b.abs().sum()) / b.numel() * 32
