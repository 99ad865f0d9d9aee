"""Attention on the GPU where single values, long sums or the order of calls matter, against its definition in 64 bits."""
import math

import pytest
import torch

import attn_ref as R
import dihydrogen_b200 as dc
from test_gpu_attention import heads
from test_gpu_ln import backend, tensor

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("queries", range(1, 10))
@pytest.mark.parametrize("masked", [False, True])
def test_infinite_values_of_the_first_keys(masked, queries, dtype):
    """Channel c holds an infinity at key c: its result is that infinity, and no other channel's is touched.  Keys about
    the tiles and parts of the kernels, of which the last is rarely full."""
    g = torch.Generator().manual_seed(21)
    be, d = backend(), 16
    for n, hq, hk, keys in ((1, 1, 1, 64), (2, 2, 1, 100), (1, 4, 2, 320), (1, 1, 1, 1001), (2, 2, 2, 4096)):
        q, k, v = (torch.randn(n, h * d, 1, c, generator=g).to(dtype) for h, c in ((hq, queries), (hk, keys), (hk, keys)))
        mask = torch.rand(n, keys, generator=g) < 0.7 if masked else torch.ones(n, keys, dtype=torch.bool)
        for b in range(n):
            there = mask[b].nonzero()[:, 0]
            for c in range(9):
                v[b, c::d, 0, there[c]] = math.inf if c % 2 else -math.inf
        want = R.attention(heads(q, hq), heads(k, hk), heads(v, hk), 1 / math.sqrt(d), kv_mask=mask, dtype=dtype)
        assert torch.isinf(want["o"][0][..., :9]).all() and torch.isfinite(want["o"][0][..., 9:]).all()
        ts = [tensor(t.cuda(), be) for t in (q, k, v)]
        o, lse = tensor(torch.full_like(q, math.nan).cuda(), be), torch.full((n, hq, queries), math.nan, device="cuda")
        dc.Attention(be, 4, hq, hk).forward(*ts, o, lse, kv_mask=mask.cuda() if masked else None)
        R.close(lse, want["lse"], "lse")
        R.close(heads(o.buffer, hq), want["o"], "o")


@pytest.mark.parametrize("queries,causal", [(8, False), (1, False), (8, True)])
def test_sums_over_a_million_keys(queries, causal):
    """Weights within 2^-10 of one another and equal values: roundings of one long running sum would all go one way
    (2.6e-4 of the result after 2^15 terms of a lane).  Heads enough that no key axis has to be cut for the SMs' sake."""
    keys, d, rows = 1 << 20, 64, 160
    heads_q = rows // queries
    g = torch.Generator(device="cuda").manual_seed(22)
    be = backend()
    q = torch.zeros(1, heads_q * d, 1, queries, device="cuda")
    q[:, ::d] = 1.0
    k = torch.zeros(1, d, 1, keys, device="cuda")
    k[:, 0] = torch.rand(1, keys, generator=g, device="cuda") * (2.0 ** -10 * math.log(2.0) * math.sqrt(d))
    v = (torch.arange(d, device="cuda", dtype=torch.float32)[:, None] * 0.1 + 0.1).expand(1, d, keys)[:, :, None].contiguous()
    o, lse = torch.full_like(q, math.nan), torch.full((1, heads_q, queries), math.nan, device="cuda")
    dc.Attention(be, 4, heads_q, 1, causal=causal).forward(*(tensor(t, be) for t in (q, k, v, o)), lse)
    s = k[0, 0, 0].double() / math.sqrt(d)
    sees = torch.arange(keys - queries + 1, keys + 1) if causal else torch.full((queries,), keys)
    want = torch.stack([torch.logsumexp(s[:int(c)], 0) for c in sees])
    # an output is a quotient of sums of the same weights: runs of at most 2^10 terms of a lane, the lanes (5), the
    # parts (2^5) and the joins' and the quotient's products, either sum
    u = 2.0 ** -24
    bound = 2 * (2 ** 10 + 5 + 2 ** 5 + 8) * u
    off = (o.reshape(heads_q, d, queries).double() / v[0, :, 0, 0].double()[:, None] - 1).abs().max()
    assert float(off) <= bound, (float(off), bound)
    # lse: its sum's roundings, those of a score (a product, scale) and its own in powers of two
    off = (lse[0].double() - want).abs().max()
    assert float(off) <= bound / 2 + 4 * u * 14, float(off)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16"])
def test_gradients_whose_offsets_pass_32_bits(dtype):
    """Keys, values and their gradients of 2^31 elements and more: equal weights, values that depend on the channel and the
    half; layer norm backward over the same memory."""
    cells, d = (1 << 25) + 40, 64
    be = backend()
    k = torch.zeros(1, d, 1, cells, dtype=dtype, device="cuda")
    v, dk, dv = (torch.empty_like(k) for _ in range(3))
    channel = torch.arange(d, device="cuda", dtype=torch.float32).to(dtype)
    v[0, :, 0, : cells // 2], v[0, :, 0, cells // 2:] = channel[:, None], -3 * channel[:, None]
    q, d_o = (torch.ones(1, d, 1, 2, dtype=dtype, device="cuda") for _ in range(2))
    o, dq, lse = torch.empty_like(q), torch.full_like(q, math.nan), torch.empty(1, 1, 2, device="cuda")
    tq, tk, tv, to, tdo, tdq, tdk, tdv = (tensor(t, be) for t in (q, k, v, o, d_o, dq, dk, dv))
    at = dc.Attention(be, 4, 1)
    at.forward(tq, tk, tv, to, lse)
    at.backward(tq, tk, tv, to, lse, tdo, tdq, tdk, tdv)
    assert at.status() == dc._abi.OK and not dq.any()
    # weights 2^-lse with lse of 25 in powers of two: three roundings of that size; of the sums 64 products each; bf16 two
    # roundings as an operand and one as a result
    rel = 3 * 25 * 2.0 ** -24 + 200 * 2.0 ** -24 + (3 * R.U16 if dtype == torch.bfloat16 else 0.0)
    for j, sign in ((0, 1), (cells // 2 - 1, 1), (cells // 2, -1), (cells - 1, -1)):
        assert float((dv[0, :, 0, j].double() * cells / 2 - 1).abs().max()) <= rel
        # two queries: scale p (d_o v - d_o o) q = (2016 + 2016) / 8 of either
        assert float((dk[0, :, 0, j].double() * cells / (sign * 1008) - 1).abs().max()) <= 2 * rel
    ln = dc.LayerNormalization(be, 4, 1e-5)
    mean, inv = ln.new_statistics(tv)
    ln.forward(tv, None, None, tdk, mean, inv)
    k[:] = (channel * channel / 64)[None, :, None, None]
    ln.backward(tv, tk, mean, inv, None, None, None, tdv)
    for j in (0, cells // 2 - 1, cells // 2, cells - 1):
        x = v[:, :, :, j].double().requires_grad_()
        y = (x - x.mean(1, keepdim=True)) / (x.var(1, keepdim=True, correction=0) + 1e-5).sqrt()
        want, = torch.autograd.grad(y, x, k[:, :, :, j].double())
        off = (dv[:, :, :, j].double() - want).abs()
        # sums of 64 terms of at most 64, an operand of inv * that
        assert bool((off <= R.stored(dtype) * want.abs() + 100 * 2.0 ** -24 * 64 * float(inv.flatten()[j])).all())
