"""Layer norm, rotary positions and attention in 64 bits on the CPU, from their definitions, each result with a bound
on what the kernels may be off by, element by element.

A rounding to bf16 is off by at most 2^-8 of the value; an fp32 sum of n products by n 2^-24 of the sum of their
magnitudes.  Where a kernel rounds weights before a product, the bound has that sum of magnitudes too."""
import math

import torch

U16, U32 = 2.0 ** -8, 2.0 ** -24


def stored(dtype):
    """The rounding of a result as it is stored."""
    return U16 if dtype == torch.bfloat16 else U32


def attention(q, k, v, scale, causal=False, q_mask=None, kv_mask=None, d_o=None, dtype=torch.float32):
    """q [n, hq, sq, d], k, v [n, hk, sk, d] as the kernels get them; {name: (value, bound)}."""
    n, hq, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    g = hq // hk
    w16 = U16 if dtype == torch.bfloat16 else 0.0  # weights and their gradients are rounded before their products
    out = stored(dtype)
    q, k, v = q.double(), k.double(), v.double()
    qm = torch.ones(n, sq, dtype=torch.bool) if q_mask is None else q_mask.bool()
    km = torch.ones(n, sk, dtype=torch.bool) if kv_mask is None else kv_mask.bool()
    zero = lambda t, m: torch.where(m[:, None, :, None], t, torch.zeros((), dtype=t.dtype))
    q, k, v = zero(q, qm), zero(k, km), zero(v, km)
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = scale * q @ kk.transpose(-1, -2)
    ok = (qm[:, None, :, None] & km[:, None, None, :]).expand(n, hq, sq, sk)
    if causal:
        ok = ok & (torch.arange(sk)[None, :] <= torch.arange(sq)[:, None] + (sk - sq))
    some = ok.any(-1, keepdim=True)
    s = torch.where(ok, s, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.where(ok & some, torch.exp(s - torch.where(some, lse, 0.0)), 0.0)
    o = p @ vv
    # a score is off by (d + 4) 2^-24 of the sum of its magnitudes, and of its own size in powers of two
    e_s = (d + 8) * U32 * scale * (q.abs() @ kk.abs().transpose(-1, -2)) + 4 * U32
    e_w = torch.where(ok, 2 * e_s.amax(-1, keepdim=True) + (sk + 16) * U32, 0.0)  # relative, of a weight
    pv = p @ vv.abs()
    e_o = ((w16 + e_w) * p) @ vv.abs() + (sk + 16) * U32 * pv
    got = {"o": (o, out * o.abs() + e_o * (1 + out)),
           "lse": (lse[..., 0], torch.where(some, e_w.amax(-1, keepdim=True) + 4 * U32 * lse.abs(), 0.0)[..., 0])}
    if d_o is None:
        return got
    do = zero(d_o.double(), qm)
    do = torch.where(some, do, 0.0)
    per = lambda t: t.reshape(n, hk, g, *t.shape[2:]).sum(2)
    dv = per(p.transpose(-1, -2) @ do)
    e_dv = per(((w16 + e_w) * p).transpose(-1, -2) @ do.abs()) + (g * sq + 16) * U32 * per(p.transpose(-1, -2) @ do.abs())
    dp = do @ vv.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # delta is taken from the stored o; dp is an fp32 sum
    e_delta = (do.abs() * got["o"][1]).sum(-1, keepdim=True) + d * U32 * (do.abs() * o.abs()).sum(-1, keepdim=True)
    e_dp = (d + 4) * U32 * (do.abs() @ vv.abs().transpose(-1, -2))
    e_ds = (w16 + e_w) * ds.abs() + p * (1 + w16) * (e_delta + e_dp + 2 * U32 * (dp.abs() + delta.abs()))
    dq, dk = scale * ds @ kk, scale * per(ds.transpose(-1, -2) @ q)
    a_q, a_k = scale * ds.abs() @ kk.abs(), scale * per(ds.abs().transpose(-1, -2) @ q.abs())
    e_dq = scale * e_ds @ kk.abs() + (sk + 16) * U32 * a_q
    e_dk = scale * per(e_ds.transpose(-1, -2) @ q.abs()) + (g * sq + 16) * U32 * a_k
    for name, x, e in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        got[name] = (x, out * x.abs() + e * (1 + out))
    return got


def layer_norm(x, scale, bias, eps, d_y=None, dtype=torch.float32):
    """x [n, c, cells] as the kernel gets it; {name: (value, bound)}."""
    out, c, cells = stored(dtype), x.shape[1], x.shape[0] * x.shape[2]
    x = x.double()
    w = torch.ones(c, dtype=torch.float64) if scale is None else scale.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    w, b = w[None, :, None], b[None, :, None]
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    inv = 1 / torch.sqrt(var + eps)
    u = (x - mean) * inv
    y = u * w + b
    top = x.abs().amax(1, keepdim=True)
    e_mean = (c + 4) * U32 * x.abs().mean(1, keepdim=True)
    # x - mean is off by e_mean and by a rounding of the difference
    e_x = e_mean + U32 * ((x - mean).abs() + top * 0)
    e_inv = (c + 16) * U32 + (e_mean * inv) ** 2 + 2 * e_mean * inv * U32 * c  # relative
    e_u = e_x * inv + u.abs() * (e_inv + 4 * U32)
    got = {"mean": (mean[:, 0], e_mean[:, 0]), "inv_std": (inv[:, 0], (inv * (e_inv + 4 * U32))[:, 0]),
           "y": (y, out * y.abs() + (e_u * w.abs() + 4 * U32 * (u * w).abs() + 2 * U32 * b.abs()) * (1 + out))}
    if d_y is None:
        return got
    g0 = d_y.double()
    g = g0 * w
    a, q = g.mean(1, keepdim=True), (g * u).mean(1, keepdim=True)
    dx = inv * (g - a - u * q)
    n32 = (c + 16) * U32
    e_a = n32 * g.abs().mean(1, keepdim=True)
    e_q = n32 * (g * u).abs().mean(1, keepdim=True) + (g.abs() * e_u).mean(1, keepdim=True)
    size = g.abs() + a.abs() + (u * q).abs()
    e_dx = inv * (e_a + e_u * q.abs() + u.abs() * e_q + 8 * U32 * size) + (e_inv + 4 * U32) * inv * size
    got["dx"] = (dx, out * dx.abs() + e_dx * (1 + out))
    got["dscale"] = ((g0 * u).sum((0, 2)), (g0.abs() * e_u).sum((0, 2)) + (cells + 16) * U32 * (g0 * u).abs().sum((0, 2)))
    got["dbias"] = (g0.sum((0, 2)), (cells + 16) * U32 * g0.abs().sum((0, 2)))
    return got


def rotary(x, head_dim, axis_channels, rotated, base, interleaved, origin, step, inverse, dtype=torch.float32):
    """x [n, c, *dims] (D outermost); axis_channels, origin, step in the order of dims; (value, bound)."""
    x = x.double()
    dims = x.shape[2:]
    y = x.clone().reshape(x.shape[0], -1, head_dim, *dims)
    src = x.reshape(y.shape)
    size = src.abs().clone()
    first = 0
    for axis, a in enumerate(axis_channels):
        where = (origin[axis] + torch.arange(dims[axis], dtype=torch.float64)) * step[axis]
        where = where.reshape([-1 if i == axis else 1 for i in range(len(dims))])
        for j in range(a // 2):
            t = where * base ** (-2.0 * j / a) * (-1 if inverse else 1)
            i0, i1 = (first + 2 * j, first + 2 * j + 1) if interleaved else (first + j, first + j + a // 2)
            p, q = src[:, :rotated, i0], src[:, :rotated, i1]
            y[:, :rotated, i0], y[:, :rotated, i1] = p * t.cos() - q * t.sin(), p * t.sin() + q * t.cos()
            size[:, :rotated, i0] = size[:, :rotated, i1] = p.abs() + q.abs()
        first += a
    out = stored(dtype)
    return y.reshape(x.shape), (out * y.abs() + 4 * U32 * size * (1 + out)).reshape(x.shape)


def close(got, want, name):
    value, bound = want
    got = got.detach().double().cpu().reshape(value.shape)
    bad = ~((got == value) | ((got - value).abs() <= bound + 1e-37))
    if bool(bad.any()):
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i]:.9g} instead of "
                             f"{value[i]:.9g}, bound {float(bound[i]):.3g}")
