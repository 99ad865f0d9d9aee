"""What the operators of attention between cells refuse, and host geometry: no GPU."""
import ctypes
import math

import pytest
import torch

import dihydrogen_b200 as dc
from dihydrogen_b200 import _abi

FAKE = 1 << 20  # an address that is checked for null and alignment only: every call here is refused before a launch


def nd(n, c, *dims, sc=None, w=1):
    d = _abi.NdDesc()
    d.nsd = len(dims)
    full = [1] * (3 - len(dims)) + list(dims)
    d.n, d.c = n, c
    cells = math.prod(full)
    d.sc = cells if sc is None else sc
    d.sn = d.sc * c
    for i, (e, s) in enumerate(zip(full, (full[1] * full[2], full[2], w))):
        d.dims[i], d.strides[i] = e, s
    return d


def status(name, *args):
    return getattr(_abi.lib(), name)(*[ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args])


def ln(xd, yd, dtype=_abi.F32, x=FAKE, eps=1e-5):
    return status("dcb_ln_fwd", xd, dtype, x, None, None, eps, yd, FAKE, None, None, None)


def test_layer_norm_refusals():
    good = nd(1, 4, 3, 5)
    assert ln(good, nd(1, 4, 3, 6)) == _abi.BAD_ARG
    assert ln(good, good, dtype=7) == _abi.BAD_ARG
    assert ln(good, good, x=None) == _abi.BAD_ARG
    assert ln(good, good, eps=-1.0) == _abi.BAD_ARG
    assert ln(good, good, eps=float("nan")) == _abi.BAD_ARG
    assert ln(nd(1, 0, 3, 5), nd(1, 0, 3, 5)) == _abi.BAD_ARG
    assert ln(nd(1, 4, 3, 5, w=2), good) == _abi.BAD_ARG  # W is not dense
    assert ln(nd(1, 16385, 1, 1), nd(1, 16385, 1, 1)) == _abi.UNSUPPORTED
    assert ln(nd(0, 4, 3, 5), nd(0, 4, 3, 5), x=None) == _abi.OK  # nothing to do
    assert status("dcb_ln_bwd_workspace_bytes", good, 3) == -1
    need = status("dcb_ln_bwd_workspace_bytes", good, _abi.BF16)
    assert need > 0
    bwd = lambda dw, db, ws, n: status("dcb_ln_bwd", good, 0, FAKE, good, FAKE, FAKE, FAKE, None, good, FAKE, dw, db, ws,
                                       n, None)
    assert bwd(FAKE, None, FAKE, need) == _abi.BAD_ARG
    assert bwd(FAKE, FAKE, None, need) == _abi.BAD_ARG
    assert bwd(FAKE, FAKE, FAKE, need - 1) == _abi.BAD_ARG
    assert bwd(FAKE, FAKE, FAKE + 4, need) == _abi.BAD_ARG


def test_layer_norm_in_place_needs_the_same_strides():
    a, b = nd(2, 4, 3, 5), nd(2, 4, 3, 5, sc=16)
    assert status("dcb_ln_fwd", a, 0, FAKE, None, None, 1e-5, b, FAKE, None, None, None) == _abi.BAD_ARG
    assert b"strides" in _abi.lib().dcb_last_error()
    for x, dy, xd, dyd in ((FAKE, 2 * FAKE, b, a), (2 * FAKE, FAKE, a, b)):
        assert status("dcb_ln_bwd", xd, 0, x, dyd, dy, FAKE, FAKE, None, a, FAKE, None, None, None, 0, None) == _abi.BAD_ARG
        assert b"strides" in _abi.lib().dcb_last_error()


def rotary(**kw):
    rd = _abi.RotaryDesc()
    rd.nsd, rd.head_dim, rd.rotated_heads, rd.base = 2, 8, 2, 100.0
    rd.axis_channels[1], rd.axis_channels[2] = 4, 4
    for i in range(3):
        rd.step[i] = 1.0
    xd = kw.pop("xd", nd(1, 24, 3, 5))
    for k, v in kw.items():
        if k == "axis":
            for i, a in enumerate(v):
                rd.axis_channels[i] = a
        else:
            setattr(rd, k, v)
    plan = ctypes.c_void_p()
    return status("dcb_rotary_plan_create", rd, xd, ctypes.byref(plan))


def test_rotary_refusals():
    for bad in (dict(head_dim=0), dict(head_dim=7), dict(rotated_heads=4), dict(rotated_heads=-1), dict(axis=(0, 3, 4)),
                dict(axis=(2, 2, 2)), dict(axis=(0, 6, 4)), dict(axis=(0, -2, 4)), dict(base=0.0),
                dict(base=float("inf")), dict(nsd=3), dict(xd=nd(1, 0, 3, 5))):
        assert rotary(**bad) == _abi.BAD_ARG, bad
    assert status("dcb_rotary_apply", None, nd(1, 8, 2, 2), 0, FAKE, nd(1, 8, 2, 2), 0, FAKE, 0, None) == _abi.BAD_ARG


def desc(q=2, kv=1, dtype=_abi.F32, scale=0.5, causal=0):
    return _abi.AttentionDesc(q, kv, dtype, causal, scale)


def attention(ad, qd, kd, vd=None, od=None, q=FAKE, lse=FAKE, ws=FAKE, size=1 << 40):
    return status("dcb_attention_fwd", ad, qd, q, kd, FAKE, vd or kd, FAKE, None, None, od or qd, FAKE, lse, ws, size,
                  None)


def test_attention_refusals():
    qd, kd = nd(1, 16, 3, 5), nd(1, 8, 4, 7)
    assert attention(desc(q=3), qd, kd) == _abi.BAD_ARG           # 16 channels are not 3 heads
    assert attention(desc(q=2, kv=0), qd, kd) == _abi.BAD_ARG
    assert attention(desc(q=2, kv=4), qd, kd) == _abi.BAD_ARG     # heads that nobody reads
    assert attention(desc(dtype=2), qd, kd) == _abi.BAD_ARG
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attention(desc(scale=scale), qd, kd) == _abi.BAD_ARG
    assert attention(desc(), qd, nd(1, 16, 4, 7)) == _abi.BAD_ARG  # heads of another size
    assert attention(desc(), qd, nd(2, 8, 4, 7)) == _abi.BAD_ARG   # samples
    assert attention(desc(), qd, kd, vd=nd(1, 8, 4, 8)) == _abi.BAD_ARG
    assert attention(desc(), qd, kd, od=nd(1, 16, 5, 3)) == _abi.BAD_ARG
    assert attention(desc(), qd, kd, q=None) == _abi.BAD_ARG
    assert attention(desc(), qd, kd, lse=None) == _abi.BAD_ARG
    assert attention(desc(), nd(1, 2 * 129, 3, 5), nd(1, 129, 4, 7)) == _abi.UNSUPPORTED
    rows = nd(1, 16, 3, 5)
    rows.strides[1] = 8  # padded rows: a shard with a halo
    assert attention(desc(), rows, kd) == _abi.UNSUPPORTED
    assert attention(desc(dtype=_abi.BF16), qd, kd, size=16) == _abi.BAD_ARG
    assert attention(desc(dtype=_abi.BF16), qd, kd, ws=None) == _abi.BAD_ARG
    assert attention(desc(dtype=_abi.BF16), qd, kd, ws=FAKE + 16) == _abi.BAD_ARG
    assert status("dcb_attention_workspace_bytes", desc(q=3), qd, kd, 0) == -1
    assert attention(desc(), nd(0, 16, 3, 5), nd(0, 8, 4, 7), q=None) == _abi.OK


def test_results_in_an_operands_place_are_refused():
    ad, qd, kd = desc(q=2, kv=1), nd(1, 16, 3, 5), nd(1, 8, 4, 7)
    far = lambda i: FAKE + (i << 20)
    for taken in range(3):
        at = [far(1), far(2), far(3)]
        assert status("dcb_attention_fwd", ad, qd, at[0], kd, at[1], kd, at[2], None, None, qd, at[taken], far(9), far(8),
                      1 << 40, None) == _abi.BAD_ARG
        assert b"place" in _abi.lib().dcb_last_error()
    names = ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv")
    for result in ("dq", "dk", "dv"):
        for other in names:
            if other == result:
                continue
            a = {n: far(i + 1) for i, n in enumerate(names)}
            a[result] = a[other]
            assert status("dcb_attention_bwd", ad, qd, a["q"], kd, a["k"], kd, a["v"], None, None, qd, a["o"], a["lse"], qd,
                          a["d_o"], qd, a["dq"], kd, a["dk"], kd, a["dv"], far(12), 1 << 40, None) == _abi.BAD_ARG
            assert b"place" in _abi.lib().dcb_last_error()


@pytest.mark.parametrize("dtype", [_abi.F32, _abi.BF16])
def test_workspaces_are_whole_units(dtype):
    """Of 256 bytes; how many depends on the parts that walks are cut in, too."""
    for cells in (1, 100, 1000, 5000, 40000):
        both = [status("dcb_attention_workspace_bytes", desc(dtype=dtype), nd(2, 128, 1, cells), nd(2, 64, 1, cells), b)
                for b in (0, 1)]
        assert both[0] % 256 == 0 and both[1] % 256 == 0
        assert 0 <= both[0] and 2 * 2 * 2 * cells * 4 <= both[1]  # the statistics at least


def tensor(shape, dtype=torch.float32, dist=None):
    loc = dc.Locale(0, 1)
    return dc.Tensor(shape, loc, dist or dc.Distribution.make_localized_distribution(len(shape)), dtype=dtype)


def test_tensors_of_16_bits():
    t = tensor([6, 4, 8, 2], torch.bfloat16)
    t.allocate("cpu")
    assert t.buffer.dtype == torch.bfloat16 and t.get_base_ptr() == t.buffer.data_ptr()
    for single in (t.desc, t.nd_desc, t.full_nd_desc, t._nd):
        with pytest.raises(TypeError):
            single()  # what the operators on single precision ask for
    with pytest.raises(TypeError):
        t.set_view(torch.zeros(2, 8, 4, 6))
    with pytest.raises(TypeError):
        tensor([6, 4, 8, 2], torch.float16)
    # rows of a shard with a halo along W: the owned cells start on 16 bytes
    t = dc.Tensor([30, 4, 3, 1], dc.Locale(0, 2), dc.Distribution.make_overlapped_distribution([2, 1, 1, 1], [1, 0, 0, 0]),
                  dtype=torch.bfloat16)
    t.allocate("cpu")
    assert t.get_pitch() % 8 == 0 and (t.get_base_ptr() - t._storage.data_ptr()) % 16 == 0


def test_channel_slices():
    t = tensor([6, 4, 8, 2], torch.bfloat16)
    t.allocate("cpu")
    s = t.channel_slice(3, 2)
    ref, ptr = s._operand()
    assert ptr == t.buffer.data_ptr() + 2 * 3 * 24 and s.local_shape == [6, 4, 2, 2]
    d = ref._obj
    assert d.c == 2 and d.n == 2 and d.sc == 24 and d.sn == 8 * 24
    for first, count in ((-1, 2), (7, 2), (0, 9)):
        with pytest.raises(ValueError):
            t.channel_slice(first, count)
    t.local_shape[-1] = 1  # fewer samples: the slice follows
    assert s.local_shape == [6, 4, 2, 1] and s._operand()[0]._obj.n == 1


def test_heads():
    class Backend:
        stream = None

    for q, kv in ((3, 2), (0, 1), (2, 0)):
        with pytest.raises(ValueError):
            dc.Attention(Backend(), 4, q, kv)
    with pytest.raises(ValueError):
        dc.LayerNormalization(Backend(), 4, -1.0)
