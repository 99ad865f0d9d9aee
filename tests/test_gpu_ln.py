"""Layer normalisation on the GPU against its definition in 64 bits (attn_ref.layer_norm)."""
import pytest
import torch

import attn_ref as R
import dihydrogen_b200 as dc

pytestmark = pytest.mark.gpu
EPS = 1e-5


def tensor(buf, be, pad=0):
    """A Tensor over a device array; `pad` shifts its start and its rows off alignment by so many elements."""
    shape = list(reversed(buf.shape))
    t = dc.Tensor(shape, be.locale, dc.Distribution.make_localized_distribution(len(shape)), dtype=buf.dtype)
    if pad:
        flat = torch.empty(buf.numel() + pad, dtype=buf.dtype, device="cuda")
        view = flat[pad:].view(buf.shape)
        view.copy_(buf)
        buf = view
    t.set_view(buf)
    return t


def backend(stream=None):
    return dc.BackendDNNLib(dc.Locale(0, 1), stream)


SHAPES = [
    (1, 1, 1, 1),          # one channel, one cell: variance 0
    (2, 3, 5, 7),
    (1, 16, 8, 8),
    (4, 16, 64, 64),
    (2, 33, 3, 9, 11),
    (1, 64, 4, 12, 20),
    (1, 100, 31, 33),
    (3, 200, 5, 6, 7),
    (1, 255, 16, 16),
    (2, 256, 7, 20),
    (1, 512, 9, 13),
    (1, 513, 4, 10),       # the kernels for many channels
    (2, 1100, 3, 5, 7),
    (1, 8, 300, 400),      # more tiles than blocks
    (1, 512, 40, 130),
]


@pytest.mark.parametrize("pad", [0, 1, 2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(shape, dtype, pad):
    g = torch.Generator().manual_seed(sum(shape))
    n, c = shape[:2]
    x = (torch.randn(shape, generator=g) * 2 + 3).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    w, b = torch.randn(c, generator=g) * 0.3 + 1, torch.randn(c, generator=g)
    be = backend()
    tx, tdy = tensor(x.cuda(), be, pad), tensor(dy.cuda(), be, pad)
    ty, tdx = tensor(torch.empty_like(x).cuda(), be, pad), tensor(torch.empty_like(x).cuda(), be, pad)
    ln = dc.LayerNormalization(be, len(shape), EPS)
    mean, inv = ln.new_statistics(tx)
    dw, db = torch.full((c,), float("nan"), device="cuda"), torch.full((c,), float("nan"), device="cuda")
    ln.forward(tx, w.cuda(), b.cuda(), ty, mean, inv)
    ln.backward(tx, tdy, mean, inv, w.cuda(), dw, db, tdx)
    want = R.layer_norm(x.flatten(2), w, b, EPS, dy.flatten(2), dtype)
    for name, got in (("y", ty.buffer), ("mean", mean), ("inv_std", inv), ("dx", tdx.buffer), ("dscale", dw),
                      ("dbias", db)):
        R.close(got, want[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_scale_bias_and_statistics_and_in_place(dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 24, 6, 10, generator=g).to(dtype)
    dy = torch.randn(2, 24, 6, 10, generator=g).to(dtype)
    be = backend()
    ln = dc.LayerNormalization(be, 4, EPS)
    want = R.layer_norm(x.flatten(2), None, None, EPS, dy.flatten(2), dtype)
    t = tensor(x.cuda(), be)
    ln.forward(t, None, None, t)
    R.close(t.buffer, want["y"], "y in place")
    t, y, d = tensor(x.cuda(), be), tensor(x.cuda(), be), tensor(dy.cuda(), be)
    mean, inv = ln.new_statistics(t)
    ln.forward(t, None, None, y, mean, inv)
    ln.backward(t, d, mean, inv, None, None, None, d)
    R.close(d.buffer, want["dx"], "dx in place")


def test_values_far_from_zero():
    """A mean that is a thousand times the spread: the variance is taken about the mean."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(1, 64, 8, 16, generator=g) + 1000.0
    be = backend()
    ln = dc.LayerNormalization(be, 4, EPS)
    t, y = tensor(x.cuda(), be), tensor(x.cuda(), be)
    mean, inv = ln.new_statistics(t)
    ln.forward(t, None, None, y, mean, inv)
    want = R.layer_norm(x.flatten(2), None, None, EPS)
    R.close(inv, want["inv_std"], "inv_std")
    R.close(y.buffer, want["y"], "y")


def test_a_nan_stays_in_its_cell():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(1, 40, 4, 50, generator=g)
    clean = x.clone()
    x[0, 7, 2, 13], x[0, 3, 1, 20] = float("nan"), float("inf")
    be = backend()
    ln = dc.LayerNormalization(be, 4, EPS)
    out = []
    for v in (x, clean):
        t, y = tensor(v.cuda(), be), tensor(v.cuda(), be)
        ln.forward(t, None, None, y)
        out.append(y.buffer.cpu())
    bad = torch.isnan(out[0])
    assert bad[0, :, 2, 13].all() and bad[0, :, 1, 20].any()
    bad[0, :, 2, 13] = bad[0, :, 1, 20] = True
    assert torch.equal(out[0][~bad], out[1][~bad])


def test_partitioned_shard_with_a_halo():
    """Owned cells only; rows apart by the halo and padded to a pitch; halo cells stay as they were."""
    g = torch.Generator().manual_seed(7)
    for dtype in (torch.float32, torch.bfloat16):
        for grid in ([2, 1, 1, 1, 1], [1, 2, 1, 1, 1], [1, 1, 2, 1, 1]):
            be = backend()
            loc = dc.Locale(1, 2)
            overlap = [1 if s > 1 else 0 for s in grid]
            dist = dc.Distribution.make_overlapped_distribution(grid, overlap)
            ts = [dc.Tensor([22, 10, 6, 20, 2], loc, dist, dtype=dtype) for _ in range(4)]
            for t in ts:
                t.allocate()
                t._storage.fill_(7.0)
            x, y, dy, dx = ts
            vx = torch.randn(x.owned().shape, generator=g).to(dtype)
            vd = torch.randn(x.owned().shape, generator=g).to(dtype)
            x.owned().copy_(vx)
            dy.owned().copy_(vd)
            ln = dc.LayerNormalization(be, 5, EPS)
            mean, inv = ln.new_statistics(x)
            w, b = torch.rand(20, generator=g) + 0.5, torch.randn(20, generator=g)
            dw, db = torch.empty(20, device="cuda"), torch.empty(20, device="cuda")
            ln.forward(x, w.cuda(), b.cuda(), y, mean, inv)
            ln.backward(x, dy, mean, inv, w.cuda(), dw, db, dx)
            want = R.layer_norm(vx.flatten(2), w, b, EPS, vd.flatten(2), dtype)
            R.close(y.owned(), want["y"], "y")
            R.close(dx.owned(), want["dx"], "dx")
            R.close(dw, want["dscale"], "dscale")
            R.close(db, want["dbias"], "dbias")
            for t in (y, dx):
                kept = t._storage.clone()
                t.owned().fill_(7.0)
                assert bool((t._storage == 7.0).all()), "cells outside the shard were written"
                del kept


def test_two_ranks_add_their_gradients_up():
    g = torch.Generator().manual_seed(8)
    x, dy = torch.randn(2, 12, 8, 24, generator=g), torch.randn(2, 12, 8, 24, generator=g)
    want = R.layer_norm(x.flatten(2), None, None, EPS, dy.flatten(2))
    total = torch.zeros(2, 12, device="cuda")
    for rank in range(2):
        be = backend()
        ts = [dc.Tensor([24, 8, 12, 2], dc.Locale(rank, 2), dc.Distribution.make_distribution([2, 1, 1, 1]))
              for _ in range(4)]
        for t in ts:
            t.allocate()
        a = slice(12 * rank, 12 * rank + 12)
        ts[0].owned().copy_(x[..., a])
        ts[1].owned().copy_(dy[..., a])
        ln = dc.LayerNormalization(be, 4, EPS)
        mean, inv = ln.new_statistics(ts[0])
        dw, db = torch.empty(12, device="cuda"), torch.empty(12, device="cuda")
        ln.forward(ts[0], None, None, ts[2], mean, inv)
        ln.backward_stage1(ts[0], ts[1], mean, inv, None, dw, db, ts[3])
        total[0] += dw
        total[1] += db
    R.close(total[0], want["dscale"], "dscale")
    R.close(total[1], want["dbias"], "dbias")


def test_gradients_against_differences():
    """The sum of dy * y moves by dx times a small step of x."""
    g = torch.Generator().manual_seed(9)
    x, dy = torch.randn(1, 10, 3, 5, generator=g), torch.randn(1, 10, 3, 5, generator=g)
    w = torch.rand(10, generator=g) + 0.5
    be = backend()
    ln = dc.LayerNormalization(be, 4, EPS)
    t, d, out = tensor(x.cuda(), be), tensor(dy.cuda(), be), tensor(x.cuda(), be)
    mean, inv = ln.new_statistics(t)
    dw, db = torch.empty(10, device="cuda"), torch.empty(10, device="cuda")
    ln.forward(t, w.cuda(), None, out, mean, inv)
    ln.backward(t, d, mean, inv, w.cuda(), dw, db, out)
    dx = out.buffer.cpu().double()
    f = lambda v: (R.layer_norm(v.flatten(2), w, None, EPS)["y"][0] * dy.flatten(2).double()).sum()
    h = 1e-5
    for at in ((0, 0, 0, 0), (0, 4, 1, 3), (0, 9, 2, 4)):
        step = torch.zeros_like(x, dtype=torch.float64)
        step[at] = h
        slope = (f(x.double() + step) - f(x.double() - step)) / (2 * h)
        # the differences' own error: third derivative times h^2, of order 1e-9 here
        assert abs(float(slope) - float(dx[at])) <= 2e-6 * float(dx.abs().max())


def test_empty_tensors_and_streams():
    be = backend()
    ln = dc.LayerNormalization(be, 4, EPS)
    ts = [tensor(torch.empty(0, 6, 3, 4, device="cuda"), be) for _ in range(3)]
    dw, db = torch.full((6,), 5.0, device="cuda"), torch.full((6,), 5.0, device="cuda")
    st = torch.empty(0, 12, device="cuda")
    ln.forward(ts[0], None, None, ts[1], st, st)
    ln.backward(ts[0], ts[1], st, st, None, dw, db, ts[2])
    assert not dw.any() and not db.any()
    # on a stream of the backend's own
    s = torch.cuda.Stream()
    be = backend(s)
    ln = dc.LayerNormalization(be, 4, EPS)
    x = torch.randn(2, 40, 16, 24)
    t, y, d, o = (tensor(x.cuda(), be) for _ in range(4))
    torch.cuda.synchronize()
    mean, inv = ln.new_statistics(t)
    dw, db = torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    ln.forward(t, None, None, y, mean, inv)
    ln.backward(t, d, mean, inv, None, dw, db, o)
    s.synchronize()
    want = R.layer_norm(x.flatten(2), None, None, EPS, x.flatten(2))
    R.close(y.buffer, want["y"], "y")
    R.close(dw, want["dscale"], "dscale")


def test_two_captured_graphs_replayed_at_once_and_the_same_bits():
    be = backend()
    ln = dc.LayerNormalization(be, 4, EPS)
    x = torch.randn(2, 48, 40, 64)
    sets = []
    for k in range(2):
        t, d, y, o = tensor(x.cuda() * (k + 1), be), tensor(x.flip(1).cuda(), be), tensor(x.cuda(), be), tensor(x.cuda(), be)
        mean, inv = ln.new_statistics(t)
        dw, db = torch.empty(48, device="cuda"), torch.empty(48, device="cuda")

        def step():
            ln.forward(t, None, None, y, mean, inv)
            ln.backward(t, d, mean, inv, None, dw, db, o)

        step()
        torch.cuda.synchronize()
        first = [v.clone() for v in (y.buffer, o.buffer, dw, db)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        sets.append((graph, first, (y.buffer, o.buffer, dw, db), (t, d, mean, inv)))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for s, (graph, *_rest) in zip(streams, sets):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _g, first, now, _k in sets:
        for a, b in zip(first, now):
            assert torch.equal(a, b)
