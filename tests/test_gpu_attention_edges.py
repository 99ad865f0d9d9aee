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
