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
