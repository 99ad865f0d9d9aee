"""Layer normalisation in 64 bits, on whatever device its inputs are, with bounds that follow the kernels' own order of
sums: they hold for every cell, also where the mean is far larger than the deviation, and are tight enough that a sum
which lost a tile of cells breaks them.

u = 2^-24 is a rounding's half step in fp32.  Of a cell with c channels, deviation s (with eps), largest |x - mean| D
and largest |x| A, all relative to the exact values of the same inputs:

* mean: sums of at most 8 values, their joins with what the rounding left carried along, a sum over at most 8 warps, each
  with a product on either side: 8 + 8 + 4 roundings of at most A.
* variance: the squares of 8 values about their own mean and of the means' differences.  m2 is a sum of ceil(c / 8)
  terms, each of at most 16 roundings; a difference of means is off by at most 16 u D (what a group's residual and the
  joins' products are rounded by), which enters twice: 32 u D / s.  What the warps' common mean is off by (12 u A at
  most) enters as its square.  inv_std is off by half of that, and by the roundings of the sum with eps, the root and
  the quotient.
* gradients of scale and bias: a thread's cells (4), the lanes (5), the tiles of a block one after the other, the groups
  of a block (8), then fp64; 3 more in the products and the last rounding.
"""
import torch

U16, U32 = 2.0 ** -8, 2.0 ** -24
WARPS, STEP = 8, 8


def launch(c, lens, runs, vec, sms, backward):
    """How a call is dealt out, as the kernels' host code chooses it: cells of a thread, warps of a group, whether a warp's
    cells lie 32 apart, tiles, blocks.  lens: cells of a run, of `runs` runs; vec: cells that one access may fetch."""
    cells = lens * runs
    four = cells >= 4 * 32 * sms
    split = four and vec < 4 and lens >= 512
    v = 4 if split or (four and vec == 4) else 1
    tiles, g = -(-cells // (32 * v)), 1
    while g < WARPS and (c > STEP * g or (c >= 2 * g and tiles * g < 8 * sms)):
        g *= 2
    groups = WARPS // g
    units = runs * (-(-lens // (32 * v)) if split else lens // v)
    per_tile = groups * (1 if split else 32)
    tiles = -(-units // per_tile)
    blocks = min(tiles, ((4 if v == 1 else 2) if backward else 4) * sms)
    return {"v": v, "g": g, "split": split, "tiles": tiles, "blocks": blocks, "partial": units % per_tile != 0 or (split and lens % (32 * v) != 0)}


def layer_norm(x, scale, bias, eps, d_y=None, tiles_a_block=1):
    """x [n, c, cells] as the kernel gets it; {name: (value, bound)}."""
    out, c = (U16 if x.dtype == torch.bfloat16 else U32), x.shape[1]
    # eps is a float to the kernels
    eps = float(torch.tensor(eps, dtype=torch.float32))
    x = x.double()
    one = lambda t, fill: torch.full((c,), fill, dtype=torch.float64, device=x.device) if t is None else t.double().to(x.device)
    w, b = one(scale, 1.0)[None, :, None], one(bias, 0.0)[None, :, None]
    mean = x.mean(1, keepdim=True)
    far = x - mean
    inv = (far.square().mean(1, keepdim=True) + eps).rsqrt()
    u = far * inv
    top, size = far.abs().amax(1, keepdim=True), x.abs().amax(1, keepdim=True)
    e_mean = 20 * U32 * size
    e_inv = (-(-c // STEP) + 16 + 32 * top * inv) / 2 * U32 + (12 * U32 * size * inv) ** 2 + 4 * U32  # relative
    e_u = inv * (e_mean + U32 * far.abs()) + u.abs() * (e_inv + 3 * U32)
    y = u * w + b
    got = {"mean": (mean[:, 0], e_mean[:, 0]), "inv_std": (inv[:, 0], (inv * e_inv)[:, 0]),
           "y": (y, out * y.abs() + (e_u * w.abs() + 2 * U32 * ((u * w).abs() + b.abs())) * (1 + out))}
    if d_y is None:
        return got
    g0 = d_y.double()
    deep = (tiles_a_block + 20) * U32
    got["dscale"] = ((g0 * u).sum((0, 2)), (g0.abs() * e_u).sum((0, 2)) + deep * (g0 * u).abs().sum((0, 2)))
    got["dbias"] = (g0.sum((0, 2)), deep * g0.abs().sum((0, 2)))
    g = g0 * w
    a, q = g.mean(1, keepdim=True), (g * u).mean(1, keepdim=True)
    dx = inv * (g - a - u * q)
    # a and q: a thread's channels one after the other, a sum over the warps
    n = (-(-c // 1) + 16) * U32
    e_a = n * g.abs().mean(1, keepdim=True)
    e_q = n * (g * u).abs().mean(1, keepdim=True) + (g.abs() * e_u).mean(1, keepdim=True)
    all_of = g.abs() + a.abs() + (u * q).abs()
    e_dx = inv * (e_a + e_u * q.abs() + u.abs() * e_q + 8 * U32 * all_of) + (e_inv + 4 * U32) * inv * all_of
    got["dx"] = (dx, out * dx.abs() + e_dx * (1 + out))
    return got
