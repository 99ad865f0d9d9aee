"""Layer normalisation on the GPU where cells lie far from zero and where blocks walk over several tiles, against its
definition in 64 bits with the bounds of ln_ref."""
import pytest
import torch

import attn_ref as R
import dihydrogen_b200 as dc
import ln_ref
from test_gpu_ln import EPS, backend, tensor

pytestmark = pytest.mark.gpu


def run(x, dy, w, b, be, tiles_a_block=1):
    """A training step on device arrays; every result is checked."""
    c = x.shape[1]
    tx, td = tensor(x, be), tensor(dy, be)
    ty, tdx = (tensor(torch.full_like(x, float("nan")), be) for _ in range(2))
    ln = dc.LayerNormalization(be, x.dim(), EPS)
    mean, inv = ln.new_statistics(tx)
    dw, db = (torch.full((c,), float("nan"), device="cuda") for _ in range(2))
    ln.forward(tx, w, b, ty, mean, inv)
    ln.backward(tx, td, mean, inv, w, dw, db, tdx)
    want = ln_ref.layer_norm(x.flatten(2), w, b, EPS, dy.flatten(2), tiles_a_block)
    for name, got in (("mean", mean), ("inv_std", inv), ("y", ty.buffer), ("dx", tdx.buffer), ("dscale", dw), ("dbias", db)):
        R.close(got, tuple(t.cpu() for t in want[name]), name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("ratio", [1, 10, 100, 1000, 10000])
@pytest.mark.parametrize("c", [3, 4, 8, 13, 16, 32, 64, 100, 513])
def test_means_far_larger_than_the_deviation(c, ratio, dtype):
    """One to eight warps a cell, full and short steps of channels; deviations of 1 and of 0.01, where eps counts; the first
    half of the channels apart from the second."""
    g = torch.Generator().manual_seed(c * ratio)
    be = backend()
    for dims, std, apart in (((50, 60), 1.0, 0.0), ((160, 200), 1.0, 3.0), ((131, 151), 0.01, 0.0)):
        x = torch.randn(1, c, *dims, generator=g) * std + ratio * std
        x[:, : c // 2] += apart * std
        dy = torch.randn(x.shape, generator=g)
        x, dy = x.to(dtype), dy.to(dtype)
        run(x.cuda(), dy.cuda(), None, None, be, 4)


# n, channels, dims, (cells of a thread, warps of a group, 32 apart) of the backward kernel on 148 SMs
MANY = [
    ((1, 8, 1100, 1000), (4, 1, False)),
    ((1, 16, 700, 900), (4, 2, False)),
    ((2, 32, 300, 602), (4, 4, False)),
    ((1, 100, 500, 500), (4, 8, False)),
    ((1, 5, 901, 701), (4, 1, True)),
    ((3, 16, 301, 401), (4, 2, True)),
    ((3, 32, 201, 301), (4, 4, True)),
    ((2, 64, 401, 301), (4, 8, True)),
    ((900, 8, 15, 33), (1, 1, False)),
    ((400, 16, 15, 33), (1, 2, False)),
    ((300, 64, 15, 33), (1, 8, False)),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape,kind", MANY, ids=lambda s: "x".join(map(str, s)))
def test_several_tiles_a_block(shape, kind, dtype):
    """Blocks of both kernels go on to further tiles, the last of which is partly empty."""
    n, c, h, w = shape
    how = {b: ln_ref.launch(c, h * w, n, 4 if h * w % 4 == 0 else 1, torch.cuda.get_device_properties(0).multi_processor_count, b)
           for b in (False, True)}
    assert (how[True]["v"], how[True]["g"], how[True]["split"]) == kind
    assert all(x["tiles"] > x["blocks"] for x in how.values()) and how[True]["partial"]
    g = torch.Generator(device="cuda").manual_seed(c)
    x = (torch.randn(shape, generator=g, device="cuda") * 2 + 0.5).to(dtype)
    dy = torch.randn(shape, generator=g, device="cuda").to(dtype)
    scale, bias = torch.rand(c, generator=g, device="cuda") + 0.5, torch.randn(c, generator=g, device="cuda")
    run(x, dy, scale, bias, backend(), -(-how[True]["tiles"] // how[True]["blocks"]))
