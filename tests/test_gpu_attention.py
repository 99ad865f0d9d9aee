"""Attention on the GPU, forward and backward, against its definition in 64 bits (attn_ref.attention)."""
import math

import pytest
import torch

import attn_ref as R
import dihydrogen_b200 as dc
from test_gpu_ln import backend, tensor

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16]
NAN = float("nan")


def heads(t, h):
    """[n, h d, dims] -> [n, h, cells, d]"""
    n = t.shape[0]
    return t.reshape(n, h, t.shape[1] // h, -1).transpose(-1, -2)


def run(n, hq, hk, d, q_dims, kv_dims, dtype, causal=False, q_mask=None, kv_mask=None, seed=0, std=1.3, pad=0, mean=0.0,
        poison=None, be=None, want_grad=True):
    """One forward and backward pass; checks everything and returns what came out."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda h, dims: (torch.randn(n, h * d, *dims, generator=g) * std + mean).to(dtype)
    q, k, v, do = rnd(hq, q_dims), rnd(hk, kv_dims), rnd(hk, kv_dims), rnd(hq, q_dims)
    want = R.attention(heads(q, hq), heads(k, hk), heads(v, hk), 1 / math.sqrt(d), causal, q_mask, kv_mask,
                       heads(do, hq) if want_grad else None, dtype)
    dev = [t.cuda() for t in (q, k, v, do)]
    if poison is not None:  # cells that are not there hold anything
        for t, m in zip(dev, (q_mask, kv_mask, kv_mask, q_mask)):
            if m is not None:
                t.flatten(2).masked_fill_(~m.bool().cuda()[:, None, :], poison)
    be = be or backend()
    tq, tk, tv, tdo = (tensor(t, be, pad) for t in dev)
    o, dq, dk, dv = (tensor(torch.full_like(t, NAN), be, pad) for t in (dev[0], dev[0], dev[1], dev[2]))
    lse = torch.full((n, hq, math.prod(q_dims)), NAN, device="cuda")
    at = dc.Attention(be, len(q_dims) + 2, hq, hk, causal=causal)
    masks = dict(q_mask=None if q_mask is None else q_mask.cuda(), kv_mask=None if kv_mask is None else kv_mask.cuda())
    at.forward(tq, tk, tv, o, lse, **masks)
    if want_grad:
        at.backward(tq, tk, tv, o, lse, tdo, dq, dk, dv, **masks)
    assert at.status() == dc.distconv._abi.OK
    assert torch.equal(torch.isneginf(lse.cpu()), torch.isneginf(want["lse"][0]))
    R.close(lse, want["lse"], "lse")
    R.close(heads(o.buffer, hq), want["o"], "o")
    if want_grad:
        R.close(heads(dq.buffer, hq), want["dq"], "dq")
        R.close(heads(dk.buffer, hk), want["dk"], "dk")
        R.close(heads(dv.buffer, hk), want["dv"], "dv")
    return o.buffer, lse, dq.buffer, dk.buffer, dv.buffer


SHAPES = [
    # n, q heads, kv heads, channels of a head, cells of q, cells of k
    (1, 1, 1, 16, (1, 1), (1, 1)),
    (2, 2, 1, 8, (1, 1), (1, 7)),
    (1, 2, 2, 32, (1, 63), (1, 65)),
    (1, 1, 1, 64, (8, 16), (8, 16)),
    (2, 4, 2, 64, (3, 5, 7), (3, 5, 7)),
    (1, 2, 1, 128, (10, 13), (10, 13)),
    (1, 3, 1, 40, (11, 12), (9, 31)),
    (2, 2, 2, 80, (4, 4, 8), (5, 5, 13)),
    (1, 8, 2, 96, (16, 20), (16, 20)),
    (1, 1, 1, 1, (4, 9), (5, 8)),
    (1, 2, 2, 7, (4, 9), (5, 8)),
    (1, 2, 2, 64, (24, 24), (24, 24)),
    (1, 2, 1, 128, (2, 150), (1, 520)),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, causal, dtype):
    run(*shape, dtype, causal=causal)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 4, 4, 64, (1, 1), (30, 70)), (2, 8, 2, 128, (1, 2), (1, 5000)),
                                   (1, 1, 1, 64, (60, 70), (1, 3)), (1, 2, 1, 32, (1, 130), (40, 101))], ids=str)
def test_few_cells_against_many(shape, dtype):
    """Long axes are split over blocks and joined."""
    run(*shape, dtype)
    run(*shape, dtype, causal=True)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("cells", [1, 2, 7, 8, 9])
def test_few_queries(cells, dtype):
    """About the counts at which another kernel takes over: channels, keys and orders off every tile, masks."""
    g = torch.Generator().manual_seed(13)
    for hq, hk, d, keys in ((4, 2, 64, 4096), (2, 2, 24, 257), (3, 1, 128, 1000), (2, 1, 33, 31), (2, 2, 65, 1336), (1, 1, 1, 8)):
        run(2, hq, hk, d, (1, cells), (1, keys), dtype)
        run(2, hq, hk, d, (1, cells), (1, keys), dtype, causal=True, pad=3)
        qm, km = torch.rand(3, cells, generator=g) < 0.7, torch.rand(3, keys, generator=g) < 0.5
        km[1], qm[2] = False, False
        run(3, hq, hk, d, (1, cells), (1, keys), dtype, q_mask=qm, kv_mask=km, poison=NAN)
        run(3, hq, hk, d, (1, cells), (1, keys), dtype, causal=True, kv_mask=km, poison=float("inf"), pad=8)
        run(3, hq, hk, d, (1, cells), (1, keys), dtype, q_mask=qm, poison=-3.3e38)


@pytest.mark.parametrize("poison", [0.0, NAN, float("inf"), -3.3e38])
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_masks(causal, dtype, poison):
    """Random masks, a sample without keys, one without queries; what masked cells hold is never seen."""
    g = torch.Generator().manual_seed(11)
    for q_dims, kv_dims, d in (((9, 17), (9, 17), 64), ((1, 200), (13, 23), 32), ((3, 4), (1, 700), 128)):
        qm = torch.rand(4, math.prod(q_dims), generator=g) < 0.7
        km = torch.rand(4, math.prod(kv_dims), generator=g) < 0.6
        km[1], qm[2] = False, False
        km[3, : km.shape[1] // 2] = False
        run(4, 2, 1, d, q_dims, kv_dims, dtype, causal=causal, q_mask=qm, kv_mask=km, poison=poison)
        run(4, 2, 1, d, q_dims, kv_dims, dtype, causal=causal, kv_mask=km, poison=poison)
        run(4, 2, 1, d, q_dims, kv_dims, dtype, causal=causal, q_mask=qm, poison=poison)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_more_queries_than_keys_under_causal_order(dtype):
    """The first cells see nothing."""
    run(2, 2, 2, 64, (1, 300), (1, 140), dtype, causal=True)
    run(1, 2, 1, 32, (1, 130), (1, 1), dtype, causal=True)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_unaligned_tensors(pad, dtype):
    run(2, 4, 2, 64, (8, 16), (8, 24), dtype, pad=pad)
    run(1, 2, 2, 72, (5, 27), (5, 27), dtype, pad=pad, causal=True)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_large_and_equal_scores(dtype):
    """Scores far from zero (the maximum is taken out), growing along the keys, and all the same."""
    run(1, 2, 2, 64, (1, 140), (1, 300), dtype, std=4.0)
    run(1, 1, 1, 16, (1, 140), (1, 300), dtype, std=0.0, mean=2.0)
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(1, 64, 1, 400, generator=g) for _ in range(3))
    k = k + torch.linspace(0, 3, 400) * q.mean(-1, keepdim=True).sign()
    q = q + q.mean(-1, keepdim=True).sign()
    be = backend()
    q, k, v = (t.to(dtype) for t in (q, k, v))
    want = R.attention(heads(q, 1), heads(k, 1), heads(v, 1), 0.125, dtype=dtype)
    ts = [tensor(t.cuda(), be) for t in (q, k, v, q)]
    lse = torch.empty(1, 1, 400, device="cuda")
    dc.Attention(be, 4, 1).forward(*ts, lse)
    R.close(heads(ts[3].buffer, 1), want["o"], "o")
    R.close(lse, want["lse"], "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_packed_projection_and_other_channels_untouched(dtype):
    """q, k and v are channels of one tensor, their gradients of another; what lies between stays."""
    g = torch.Generator().manual_seed(5)
    n, hq, hk, d, dims = 2, 4, 2, 32, (6, 22)
    qkv = torch.randn(n, (hq + 2 * hk) * d + 5, *dims, generator=g).to(dtype)
    do = torch.randn(n, hq * d, *dims, generator=g).to(dtype)
    be = backend()
    t, dt = tensor(qkv.cuda(), be), tensor(torch.full_like(qkv, 3.0).cuda(), be)
    o, tdo = tensor(torch.empty_like(do).cuda(), be), tensor(do.cuda(), be)
    lse = torch.empty(n, hq, 132, device="cuda")
    cut = lambda x: (x.channel_slice(5, hq * d), x.channel_slice(5 + hq * d, hk * d),
                     x.channel_slice(5 + (hq + hk) * d, hk * d))
    at = dc.Attention(be, 4, hq, hk)
    at.forward(*cut(t), o, lse)
    at.backward(*cut(t), o, lse, tdo, *cut(dt))
    q, k, v = qkv[:, 5:].split([hq * d, hk * d, hk * d], 1)
    want = R.attention(heads(q, hq), heads(k, hk), heads(v, hk), 1 / math.sqrt(d), d_o=heads(do, hq), dtype=dtype)
    R.close(heads(o.buffer, hq), want["o"], "o")
    assert bool((dt.buffer[:, :5] == 3.0).all())
    dq, dk, dv = dt.buffer[:, 5:].split([hq * d, hk * d, hk * d], 1)
    for name, x, h in (("dq", dq, hq), ("dk", dk, hk), ("dv", dv, hk)):
        R.close(heads(x, h), want[name], name)


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(6)
    q, k, v, do = (torch.randn(1, 16, 3, 7, generator=g) for _ in range(4))
    be = backend()
    ts = [tensor(t.cuda(), be) for t in (q, k, v, do)]
    o, dq, dk, dv = (tensor(torch.empty_like(q).cuda(), be) for _ in range(4))
    lse = torch.empty(1, 2, 21, device="cuda")
    at = dc.Attention(be, 4, 2)
    at.forward(*ts[:3], o, lse)
    at.backward(*ts[:3], o, lse, ts[3], dq, dk, dv)

    def f(*x):
        return (R.attention(*[heads(t, 2) for t in x], 8 ** -0.5)["o"][0] * heads(do, 2).double()).sum()

    h, x = 1e-5, [t.double() for t in (q, k, v)]
    for which, grad in enumerate((dq, dk, dv)):
        for at_ in ((0, 0, 0, 0), (0, 9, 2, 3), (0, 15, 1, 6)):
            step = torch.zeros_like(x[0])
            step[at_] = h
            up = [t + step if i == which else t for i, t in enumerate(x)]
            down = [t - step if i == which else t for i, t in enumerate(x)]
            slope = float(f(*up) - f(*down)) / (2 * h)
            have = grad.buffer.cpu().double()
            assert abs(slope - float(have[at_])) <= 1e-5 * float(have.abs().max())


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_the_same_bits_every_run_on_streams_and_in_graphs(dtype):
    shape = dict(n=2, hq=4, hk=2, d=64, q_dims=(9, 31), kv_dims=(9, 31))
    first = [t.clone() for t in run(*shape.values(), dtype)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    again = run(*shape.values(), dtype, be=backend(s))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))

    g = torch.Generator().manual_seed(8)
    be = backend()
    sets = []
    for k in range(2):
        q, kk, v, do = (tensor((torch.randn(1, 128, 1, c, generator=g)).to(dtype).cuda(), be) for c in (40, 900, 900, 40))
        o, dq, dk, dv = (tensor(torch.empty_like(t.buffer), be) for t in (q, q, kk, v))
        lse = torch.empty(1, 2, 40, device="cuda")
        at = dc.Attention(be, 4, 2)

        def step():
            at.forward(q, kk, v, o, lse)
            at.backward(q, kk, v, o, lse, do, dq, dk, dv)

        step()
        torch.cuda.synchronize()
        out = [t.buffer for t in (o, dq, dk, dv)] + [lse]
        want = [t.clone() for t in out]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        sets.append((graph, out, want, (q, kk, v, do)))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                x[0].replay()
    torch.cuda.synchronize()
    for _g, out, want, _k in sets:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
def test_a_captured_query_replayed_with_other_inputs(masked, dtype):
    """Two graphs of one layer replayed at once on two streams, then again: what they read is what is there now."""
    be, g = backend(), torch.Generator().manual_seed(16)
    layer, graphs = dc.Attention(be, 4, 4, 2), []
    for keys in (5000, 777):
        q, k, v = (torch.zeros(2, h * 64, 1, c, dtype=dtype, device="cuda") for h, c in ((4, 1), (2, keys), (2, keys)))
        o, lse = torch.zeros_like(q), torch.zeros(2, 4, 1, device="cuda")
        mask = torch.ones(2, keys, dtype=torch.uint8, device="cuda") if masked else None
        args = (*(tensor(t, be) for t in (q, k, v, o)), lse)
        layer.forward(*args, kv_mask=mask)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.forward(*args, kv_mask=mask)
        graphs.append((graph, torch.cuda.Stream(), q, k, v, o, lse, mask))
    for _ in range(3):
        want = []
        for _, _, q, k, v, _, _, mask in graphs:
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g))
            if masked:
                mask.copy_(torch.rand(mask.shape, generator=g) < 0.7)
            host = [t.cpu() for t in (q, k, v)]
            want.append(R.attention(heads(host[0], 4), heads(host[1], 2), heads(host[2], 2), 0.125,
                                    kv_mask=mask.cpu() if masked else None, dtype=dtype))
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, _, o, lse, _), w in zip(graphs, want):
            R.close(lse, w["lse"], "lse")
            R.close(heads(o, 4), w["o"], "o")


def test_masks_of_many_cells():
    """A mask is counted in parts of 8192 cells and more, from any address; any byte that is not zero counts."""
    g = torch.Generator().manual_seed(15)
    for keys, first in ((8192, 0), (8193, 1), (40001, 5), (64 * 8192 + 7, 3)):
        km = (torch.rand(2, keys, generator=g) < 0.3).to(torch.uint8) * torch.randint(1, 256, (2, keys), generator=g).to(torch.uint8)
        km[0, : keys // 2] = 0
        q, k, v = (torch.randn(2, 16, 1, c, generator=g) for c in (3, keys, keys))
        want = R.attention(heads(q, 2), heads(k, 2), heads(v, 2), 1 / math.sqrt(8), kv_mask=km)
        be = backend()
        room = torch.zeros(2 * keys + first, dtype=torch.uint8, device="cuda")
        mask = room[first:].view(2, keys)
        mask.copy_(km)
        tq, tk, tv = (tensor(t.cuda(), be) for t in (q, k, v))
        o, lse = tensor(torch.full_like(q, NAN).cuda(), be), torch.full((2, 2, 3), NAN, device="cuda")
        dc.Attention(be, 4, 2, 2).forward(tq, tk, tv, o, lse, kv_mask=mask)
        R.close(lse, want["lse"], "lse")
        R.close(heads(o.buffer, 2), want["o"], "o")


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("queries", [1, 6, 150])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_a_key_that_is_not_a_number_reaches_the_queries_that_see_it(d, queries, dtype):
    g = torch.Generator().manual_seed(14)
    be = backend()
    keys = 150
    for bad in (0, 13, 14, 15, 30, 63, 64, 127, 149):
        for causal in (False, True):
            q, k, v = (torch.randn(1, d, 1, c, generator=g).to(dtype).cuda() for c in (queries, keys, keys))
            k[..., bad] = NAN
            o, lse = torch.zeros_like(q), torch.zeros(1, 1, queries, device="cuda")
            dc.Attention(be, 4, 1, 1, causal=causal).forward(*(tensor(t, be) for t in (q, k, v, o)), lse)
            sees = torch.arange(queries) + (keys - queries if causal else keys) >= bad
            assert torch.equal(lse.flatten().isnan().cpu(), sees)
            assert torch.equal(o.isnan().all(1).flatten().cpu(), sees) and torch.equal(o.isnan().any(1).flatten().cpu(), sees)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_empty_sides(dtype):
    be = backend()
    at = dc.Attention(be, 4, 2)
    e = lambda c: tensor(torch.full((2, 32, 1, c), 5.0, device="cuda").to(dtype), be)
    q, k, o, dq, dk, dv = e(9), e(0), e(9), e(9), e(0), e(0)
    lse = torch.zeros(2, 2, 9, device="cuda")
    at.forward(q, k, k, o, lse)
    assert not o.buffer.any() and bool(torch.isneginf(lse).all())
    at.backward(q, k, k, o, lse, o, dq, dk, dv)
    assert not dq.buffer.any()
    q, k, dk, dv = e(0), e(9), e(9), e(9)
    lse = torch.zeros(2, 2, 0, device="cuda")
    at.forward(q, k, k, q, lse)
    at.backward(q, k, k, q, lse, q, q, dk, dv)
    assert not dk.buffer.any() and not dv.buffer.any()


def test_a_block_of_a_network():
    """Layer norm, projection by a 1 x 1 convolution, rotary positions, attention, and all their gradients."""
    torch.manual_seed(0)
    n, c, h, d, dims = 1, 16, 2, 16, (12, 20)
    be = backend()
    x, w = torch.randn(n, c, *dims), torch.randn(3 * h * d, c, 1, 1) / 4
    dy = torch.randn(n, h * d, *dims)
    gamma, beta = torch.rand(c) + 0.5, torch.randn(c)
    new = lambda ch, dtype=torch.float32: tensor(torch.empty(n, ch, *dims, dtype=dtype, device="cuda"), be)
    tx, u, du, dx = tensor(x.cuda(), be), new(c), new(c), new(c)
    qkv, dqkv = new(3 * h * d), new(3 * h * d)
    r, dr, o = new(3 * h * d, torch.bfloat16), new(3 * h * d, torch.bfloat16), new(h * d, torch.bfloat16)
    tdo = tensor(dy.bfloat16().cuda(), be)
    wt, dw = w.cuda(), torch.empty_like(w).cuda()
    gc, bc, dg, db = gamma.cuda(), beta.cuda(), torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    ln, rot, at = dc.LayerNormalization(be, 4, 1e-5), dc.RotaryPositions(be, 4), dc.Attention(be, 4, h)
    conv = dc.Convolution(be, 4)
    conv.setup(u, wt, qkv, du, dw, dqkv, [0, 0], [1, 1], [1, 1])
    rot.setup(qkv, d, [8, 8], rotated_heads=2 * h)
    mean, inv = ln.new_statistics(tx)
    lse = torch.empty(n, h, 240, device="cuda")
    cut = lambda t: [t.channel_slice(i * h * d, h * d) for i in range(3)]
    ln.forward(tx, gc, bc, u, mean, inv)
    conv.forward(1.0, u, wt, 0.0, qkv)
    rot.forward(qkv, r)
    at.forward(*cut(r), o, lse)
    at.backward(*cut(r), o, lse, tdo, *cut(dr))
    rot.backward(dr, dqkv)
    conv.backward_data(1.0, wt, dqkv, 0.0, du)
    conv.backward_filter(1.0, u, dqkv, 0.0, dw)
    ln.backward(tx, du, mean, inv, gc, dg, db, dx)
    assert at.status() == dc.distconv._abi.OK

    leaves = [t.double().requires_grad_() for t in (x, gamma, beta, w)]
    lx, lg, lb, lw = leaves
    m = lx.mean(1, keepdim=True)
    un = (lx - m) / torch.sqrt(((lx - m) ** 2).mean(1, keepdim=True) + 1e-5) * lg[None, :, None, None] + lb[None, :, None, None]
    proj = torch.einsum("kc,ncyx->nkyx", lw[:, :, 0, 0], un).reshape(n, 3, h, d, *dims)
    parts = []
    for i in range(3):
        t = proj[:, i]
        if i < 2:
            out = []
            for axis, first in ((0, 0), (1, 8)):
                pos = torch.arange(dims[axis], dtype=torch.float64).reshape((-1, 1) if axis == 0 else (1, -1))
                ang = torch.stack([pos * 10000.0 ** (-2.0 * j / 8) for j in range(4)]).expand(4, *[s if k == axis else 1 for k, s in enumerate(dims)])
                p, q = t[:, :, first:first + 4], t[:, :, first + 4:first + 8]
                out += [p * ang.cos() - q * ang.sin(), p * ang.sin() + q * ang.cos()]
            t = torch.cat(out, 2)
        parts.append(t.reshape(n, h, d, -1).transpose(-1, -2))
    q, k, v = parts
    y = torch.softmax(q @ k.transpose(-1, -2) / 4.0, -1) @ v
    y.backward(dy.bfloat16().double().reshape(n, h, d, -1).transpose(-1, -2))
    # q, k, v (2^-8 each), weights, o, and the gradients' roundings: eight roundings of 2^-8 in the norm, each at most
    # carried over once with a factor of about 1
    rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())
    assert rel(heads(o.buffer, h), y.detach()) < 8 * 2 ** -8
    for got, leaf in ((dx.buffer, lx), (dg, lg), (db, lb), (dw, lw)):
        assert rel(got.reshape(leaf.shape), leaf.grad) < 8 * 2 ** -8


def test_calls_that_are_refused():
    be = backend()
    at = dc.Attention(be, 4, 2, 1)
    t = lambda c, cells=12, dtype=torch.float32: tensor(torch.zeros(1, c, 1, cells, dtype=dtype, device="cuda"), be)
    q, k, lse = t(16), t(8), torch.zeros(1, 2, 12, device="cuda")
    bad = [
        (t(16), t(16), t(16), q, lse, {}),                                  # heads of another size
        (q, k, t(8, 11), q, lse, {}),                                       # v has other cells
        (q, t(8, dtype=torch.bfloat16), t(8, dtype=torch.bfloat16), q, lse, {}),
        (q, k, k, t(16, 11), lse, {}),
        (q, k, k, q, lse[:, :1], {}),
        (q, k, k, q, lse.double(), {}),
        (q, k, k, q, lse.cpu(), {}),
        (q, k, k, q, None, {}),
        (q, k, k, q, lse, {"kv_mask": torch.ones(1, 11, dtype=torch.bool, device="cuda")}),
        (q, k, k, q, lse, {"q_mask": torch.ones(1, 12, device="cuda")}),
        (q, k, k, q, lse, {"q_mask": torch.ones(1, 24, dtype=torch.bool, device="cuda")[:, ::2]}),
    ]
    for *args, kw in bad:
        with pytest.raises(ValueError):
            at.forward(*args, **kw)
    with pytest.raises(ValueError):
        dc.Attention(be, 4, 2, 2).forward(t(258), t(258), t(258), t(258), lse)  # 129 channels a head
    part = dc.Tensor([12, 4, 16, 1], dc.Locale(0, 2), dc.Distribution.make_distribution([2, 1, 1, 1]))
    part.allocate()
    with pytest.raises(ValueError):
        at.forward(part, part, part, part, lse)
    ln = dc.LayerNormalization(be, 4, 1e-5)
    with pytest.raises(ValueError):
        ln.forward(q, torch.ones(16), None, q)  # scale on the host
    with pytest.raises(ValueError):
        ln.forward(q, torch.ones(15, device="cuda"), None, q)
    with pytest.raises(ValueError):
        ln.backward(q, q, None, None, None, None, None, q)
    rot = dc.RotaryPositions(be, 4)
    rot.setup(q, 8, [4, 4])
    with pytest.raises(ValueError):
        rot.forward(k, k)
    with pytest.raises(dc.distconv._abi.DcbError):
        rot.setup(q, 8, [3, 4])


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_offsets_that_pass_32_bits(dtype):
    """Keys and values of 2^31 elements and more: weights are equal, values depend on the channel and the half."""
    cells, d = (1 << 25) + 40, 64
    be = backend()
    k = torch.zeros(1, d, 1, cells, dtype=dtype, device="cuda")
    v = torch.empty_like(k)
    channel = torch.arange(d, device="cuda", dtype=torch.float32).to(dtype)
    v[0, :, 0, : cells // 2], v[0, :, 0, cells // 2:] = channel[:, None], -3 * channel[:, None]
    q, o = torch.ones(1, d, 1, 2, dtype=dtype, device="cuda"), torch.empty(1, d, 1, 2, dtype=dtype, device="cuda")
    lse = torch.empty(1, 1, 2, device="cuda")
    at = dc.Attention(be, 4, 1)
    at.forward(*(tensor(t, be) for t in (q, k, v, o)), lse)
    # o = -channel: sums of equal weights, in parts of at most 2^25 terms
    want = -torch.arange(d, dtype=torch.float64)[:, None].expand(d, 2)
    off = (o[0, :, 0].double().cpu() - want).abs().max()
    assert float(off) <= 64 * (R.stored(dtype) + 2.0 ** -10), float(off)
    assert float((lse.double().cpu() - math.log(cells)).abs().max()) < 1e-3
    # and the other operators over the same memory
    tv, tk = tensor(v, be), tensor(k, be)
    ln = dc.LayerNormalization(be, 4, 1e-5)
    ln.forward(tv, None, None, tk)
    u = (channel.double() - channel.double().mean()) / channel.double().std(correction=0)
    for j, sign in ((0, 1), (cells - 1, -1)):
        assert float((k[0, :, 0, j].double() - sign * u).abs().max()) <= 2 * R.stored(dtype) * 2 + 1e-4
    rot = dc.RotaryPositions(be, 4)
    rot.setup(tv, d, [0, 2])
    rot.forward(tv, tk)
    assert torch.equal(k[0, 2:, 0, -5:], v[0, 2:, 0, -5:])


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_two_calls_at_once(dtype):
    """Two layers on two streams, masked and not, many times: neither sees the other's workspace."""
    g = torch.Generator().manual_seed(12)
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for s in streams:
        be = backend(s)
        q, k, v, do = (tensor(torch.randn(2, 64, 9, 15, generator=g).to(dtype).cuda(), be) for _ in range(4))
        o, dq, dk, dv = (tensor(torch.empty_like(q.buffer), be) for _ in range(4))
        lse = torch.empty(2, 2, 135, device="cuda")
        mask = (torch.rand(2, 135, generator=g) < 0.7).cuda()
        at = dc.Attention(be, 4, 2)

        def step(at=at, q=q, k=k, v=v, o=o, lse=lse, do=do, dq=dq, dk=dk, dv=dv, mask=mask):
            at.forward(q, k, v, o, lse, q_mask=mask, kv_mask=mask)
            at.backward(q, k, v, o, lse, do, dq, dk, dv, q_mask=mask, kv_mask=mask)

        torch.cuda.synchronize()
        step()
        torch.cuda.synchronize()
        out = [o.buffer, dq.buffer, dk.buffer, dv.buffer, lse]
        sets.append((step, out, [t.clone() for t in out]))
    torch.cuda.synchronize()
    for _ in range(20):
        for step, *_ in sets:
            step()
    torch.cuda.synchronize()
    for _s, out, want in sets:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
