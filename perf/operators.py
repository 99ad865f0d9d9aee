"""Operators of attention over the cells of an image or a volume, as cases that can be timed.

* ``norm``       layer norm over the channels of every cell (``LayerNormalization``)
* ``rotary``     rotary positions along D, H and W (``RotaryPositions``): the queries' and keys' channels of a
                 packed projection are turned, the values' are passed on; ``to`` is the type that comes out
* ``attention``  scaled dot-product attention between cells (``Attention``), ``train`` with its backward pass

Tensors are NC[D]HW: a cell's channels lie a whole volume apart, a channel's cells are contiguous.  ``dims`` is
"DxHxW" or "HxW".  An attention whose ``q_dims`` and ``kv_dims`` are equal takes its queries, keys and values out of
one packed projection, as a 1 x 1 x 1 convolution leaves them; otherwise keys and values are packed alone.  ``mask``:
only a box of every sample's cells is there, as in a batch of volumes of several extents.
"""
import math

import torch

own = False

EPS = 1e-5
BASE = 10000.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _norm(name, do, n, c, dims, dtype):
    case = {"op": "norm", "do": do, "n": n, "c": c, "dims": dims, "dtype": dtype}
    return dict(case, name=name) if name else case


def _rotary(name, do, n, q_heads, kv_heads, head_dim, dims, dtype, to):
    case = {"op": "rotary", "do": do, "n": n, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dims": dims, "dtype": dtype, "to": to}
    return dict(case, name=name) if name else case


def _attention(name, do, n, q_heads, kv_heads, head_dim, q_dims, kv_dims, dtype, causal=False, mask=False):
    case = {"op": "attention", "do": do, "n": n, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "q_dims": q_dims, "kv_dims": kv_dims, "dtype": dtype, "causal": causal, "mask": mask}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the 2-D layer of the reference's CPU example, a training step: a megabyte, where launches count
        _norm("norm2d_64_train", "train", 4, 16, "64x64", "f32"),
        # a volume inside a network, a training step in single precision
        _norm("norm3d_96_train", "train", 1, 64, "96x96x96", "f32"),
        # a cropped volume, two samples, no extent a multiple of anything, stored in 16 bits: a serving step
        _norm("norm3d_ragged_bf16", "forward", 2, 200, "19x37x53", "bf16"),
        # the projection of a small image's cells, rounded to 16 bits on its way to the attention
        _rotary("rotary2d_64", "forward", 1, 8, 8, 64, "64x64", "f32", "bf16"),
        # the gradient of a volume's projection, all in 16 bits
        _rotary("rotary3d_40_grad", "backward", 2, 8, 2, 128, "40x40x40", "bf16", "bf16"),
        # odd extents in single precision, gradient
        _rotary("rotary3d_ragged_grad", "backward", 1, 4, 2, 48, "23x37x41", "f32", "f32"),
        # pooling by attention: one query a sample reads a whole volume
        _attention("pool_query_32", "forward", 2, 8, 8, 64, "1x1", "32x32x32", "bf16"),
        # serving the network of images: a whole image's cells, 4 samples
        _attention("image64", "forward", 4, 8, 8, 64, "64x64", "64x64", "bf16"),
        # a small volume in single precision, odd extents, some cells missing
        _attention("volume_ragged_f32", "train", 1, 4, 4, 32, "9x11x13", "9x11x13", "f32", mask=True),
        # training on images
        _attention("image64_train", "train", 2, 8, 8, 64, "64x64", "64x64", "bf16"),
        # training on cropped volumes of several extents: shared keys, odd extents, cells missing
        _attention("volume_ragged_train", "train", 2, 8, 2, 80, "13x17x19", "13x17x19", "bf16", mask=True),
        # training a model that predicts a volume cell by cell
        _attention("volume_causal_train", "train", 1, 8, 2, 128, "16x24x32", "16x24x32", "bf16", causal=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _dims(rng, cells, nsd=None):
    """Extents of about so many cells."""
    nsd = nsd or rng.choice((2, 3))
    side = cells ** (1.0 / nsd)
    ext = [max(1, int(side * math.exp(rng.uniform(-0.4, 0.4)))) for _ in range(nsd - 1)]
    ext.append(max(1, int(cells / math.prod(ext))))
    if rng.random() < 0.4:  # aligned, as most networks have them
        ext[-1] = max(8, ext[-1] // 8 * 8)
    return "x".join(str(e) for e in ext)


def draw(rng):
    op = rng.choice(("norm", "rotary", "attention", "attention"))
    if op == "norm":
        n, c = rng.choice((1, 2, 4)), _spread(rng, 4, 512)
        cells = _spread(rng, 64, 50_000_000 // (n * c))
        return _norm(None, rng.choice(("forward", "train")), n, c, _dims(rng, cells), rng.choice(("f32", "bf16")))
    kv_heads = rng.choice((1, 2, 4, 8))
    q_heads = kv_heads * rng.choice((1, 1, 2, 4))
    if op == "rotary":
        n, head_dim = rng.choice((1, 2)), rng.choice((16, 32, 48, 64, 96, 128))
        cells = _spread(rng, 64, 50_000_000 // (n * (q_heads + 2 * kv_heads) * head_dim))
        dtype, to = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")))
        return _rotary(None, rng.choice(("forward", "backward")), n, q_heads, kv_heads, head_dim, _dims(rng, cells),
                       dtype, to)
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    n, head_dim = rng.choice((1, 2, 3)), rng.choice((16, 32, 40, 64, 64, 80, 96, 128, 128))
    most = (400_000_000 if dtype == "bf16" else 40_000_000) // (n * q_heads)  # pairs of one head
    kind = rng.choice(("self", "self", "self", "cross", "query"))
    if kind == "self":
        q_dims = kv_dims = _dims(rng, _spread(rng, 16, min(12288, math.isqrt(most))))
    else:
        kv = _spread(rng, 16, 40000)
        kv_dims = _dims(rng, kv)
        q_dims = _dims(rng, 1 if kind == "query" else _spread(rng, 2, min(8192, max(2, most // kv))))
        if q_dims == kv_dims:
            kv_dims = "5x7x11"
    return _attention(None, rng.choice(("forward", "train")), n, q_heads, kv_heads, head_dim, q_dims, kv_dims, dtype,
                      causal=kind == "self" and rng.random() < 0.3, mask=rng.random() < 0.3)


def _ext(dims):
    return [int(v) for v in dims.split("x")]


def _cells(dims):
    return math.prod(_ext(dims))


def _axis_channels(head_dim, nsd):
    """Channels of a head that D, H and W turn: about a third (half) each, even."""
    part = head_dim // nsd // 2 * 2
    return [0] * (3 - nsd) + [part] * (nsd - 1) + [(head_dim - part * (nsd - 1)) // 2 * 2]


def _box(dims, sample):
    """The cells of a sample that are there."""
    ext = _ext(dims)
    keep = torch.zeros(ext, dtype=torch.bool)
    keep[tuple(slice(0, max(1, e - e // 4 - sample % 3)) for e in ext)] = True
    return keep.reshape(-1)


def _masks(case):
    """Which cells are there: of the queries' grid (only where it is the keys' too) and of the keys'."""
    if not case["mask"]:
        return None, None
    kv = torch.stack([_box(case["kv_dims"], i) for i in range(case["n"])])
    return (kv if case["q_dims"] == case["kv_dims"] else None), kv


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op, n = case["op"], case["n"]

    def normal(shape, dtype, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)

    def empty(shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=dev)

    s = {"case": dict(case)}
    if op == "norm":
        t, shape = TYPES[case["dtype"]], (n, case["c"], *_ext(case["dims"]))
        s.update(x=normal(shape, t, 2.0, 0.5), scale=normal(case["c"], torch.float32, 0.2, 1.0),
                 bias=normal(case["c"], torch.float32, 0.2), y=empty(shape, t),
                 mean=empty((n, _cells(case["dims"]))), inv_std=empty((n, _cells(case["dims"]))))
        if case["do"] == "train":
            s.update(d_y=normal(shape, t), d_x=empty(shape, t), d_scale=empty(case["c"]), d_bias=empty(case["c"]))
    elif op == "rotary":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        shape = (n, heads * case["head_dim"], *_ext(case["dims"]))
        a, b = TYPES[case["dtype"]], TYPES[case["to"]]
        if case["do"] == "forward":
            s.update(x=normal(shape, a), y=empty(shape, b))
        else:  # the gradient comes in the type that went out
            s.update(x=normal(shape, b), y=empty(shape, a))
    else:
        t, d = TYPES[case["dtype"]], case["head_dim"]
        q_ext, kv_ext = _ext(case["q_dims"]), _ext(case["kv_dims"])
        q_ch, kv_ch = case["q_heads"] * d, 2 * case["kv_heads"] * d
        packed = case["q_dims"] == case["kv_dims"]
        if packed:
            s["qkv"] = normal((n, q_ch + kv_ch, *q_ext), t, 1.3)
        else:
            s["q"], s["kv"] = normal((n, q_ch, *q_ext), t, 1.3), normal((n, kv_ch, *kv_ext), t, 1.3)
        s["q_mask"], s["kv_mask"] = (m if m is None else m.to(dev) for m in _masks(case))
        s["o"], s["lse"] = empty((n, q_ch, *q_ext), t), empty((n, case["q_heads"], _cells(case["q_dims"])))
        if case["do"] == "train":
            s["d_o"] = normal((n, q_ch, *q_ext), t)
            for name in ("qkv",) if packed else ("q", "kv"):
                s["d_" + name] = empty(s[name].shape, t)
    if own:
        s["own"] = _handles(case, s)
    return s


# ---- the framework's operators -------------------------------------------------------------------------------------


def _handles(case, s):
    """The layer and the tensors that a program keeps over the buffers above."""
    import dihydrogen_b200 as dc

    be = dc.BackendDNNLib(dc.Locale(0, 1))

    def tensor(buf):
        shape = list(reversed(buf.shape))
        t = dc.Tensor(shape, be.locale, dc.Distribution.make_localized_distribution(len(shape)), dtype=buf.dtype)
        t.set_view(buf)
        return t

    h = {k: tensor(s[k]) for k in ("x", "y", "d_x", "d_y", "q", "kv", "qkv", "o", "d_o", "d_q", "d_kv", "d_qkv")
         if k in s}
    if case["op"] == "norm":
        h["layer"] = dc.LayerNormalization(be, h["x"].get_num_dims(), EPS)
    elif case["op"] == "rotary":
        nd = h["x"].get_num_dims()
        h["layer"] = dc.RotaryPositions(be, nd)
        h["layer"].setup(h["x"], case["head_dim"], list(reversed(_axis_channels(case["head_dim"], nd - 2)))[:nd - 2],
                         rotated_heads=case["q_heads"] + case["kv_heads"], base=BASE)
    else:
        q_ch, kv_ch = case["q_heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        for p in ("", "d_"):
            if p + "qkv" in h:
                t = h[p + "qkv"]
                h[p + "qkv3"] = (t.channel_slice(0, q_ch), t.channel_slice(q_ch, kv_ch),
                                 t.channel_slice(q_ch + kv_ch, kv_ch))
            elif p + "q" in h:
                t = h[p + "kv"]
                h[p + "qkv3"] = (h[p + "q"], t.channel_slice(0, kv_ch), t.channel_slice(kv_ch, kv_ch))
        h["layer"] = dc.Attention(be, h["o"].get_num_dims(), case["q_heads"], case["kv_heads"], causal=case["causal"])
    return h


def _run_own(s):
    case, h = s["case"], s["own"]
    layer = h["layer"]
    if case["op"] == "norm":
        layer.forward(h["x"], s["scale"], s["bias"], h["y"], s["mean"], s["inv_std"])
        if case["do"] == "train":
            layer.backward(h["x"], h["d_y"], s["mean"], s["inv_std"], s["scale"], s["d_scale"], s["d_bias"], h["d_x"])
    elif case["op"] == "rotary":
        (layer.forward if case["do"] == "forward" else layer.backward)(h["x"], h["y"])
    else:
        layer.forward(*h["qkv3"], h["o"], s["lse"], q_mask=s["q_mask"], kv_mask=s["kv_mask"])
        if case["do"] == "train":
            layer.backward(*h["qkv3"], h["o"], s["lse"], h["d_o"], *h["d_qkv3"], q_mask=s["q_mask"],
                           kv_mask=s["kv_mask"])
    return {k: s[k] for k in ("y", "mean", "inv_std", "d_x", "d_scale", "d_bias", "o", "lse", "d_qkv", "d_q", "d_kv")
            if k in s}


# ---- their plain form ----------------------------------------------------------------------------------------------


def _plain_norm(case, s):
    t, c = s["x"].dtype, case["c"]
    per_channel = (1, c) + (1,) * (s["x"].dim() - 2)
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    inv_std = (centred.square().mean(1, keepdim=True) + EPS).rsqrt()
    unit = centred * inv_std
    got = {"y": (unit * s["scale"].view(per_channel) + s["bias"].view(per_channel)).to(t),
           "mean": mean.reshape(case["n"], -1), "inv_std": inv_std.reshape(case["n"], -1)}
    if case["do"] == "train":
        d_y = s["d_y"].float()
        over = [i for i in range(x.dim()) if i != 1]
        by_unit = d_y * s["scale"].view(per_channel)
        got["d_x"] = ((by_unit - by_unit.mean(1, keepdim=True) - unit * (by_unit * unit).mean(1, keepdim=True))
                      * inv_std).to(t)
        got["d_scale"], got["d_bias"] = (d_y * unit).sum(over), d_y.sum(over)
    return got


def _angles(case, device):
    """Angle of every pair of channels at every cell, [pairs, cells], in 64 bits: the pairs of D, then H, then W."""
    ext = _ext(case["dims"])
    parts = _axis_channels(case["head_dim"], len(ext))[3 - len(ext):]
    where = torch.meshgrid(*[torch.arange(e, device=device, dtype=torch.float64) for e in ext], indexing="ij")
    return [p.reshape(1, -1) * (BASE ** (-torch.arange(0, a, 2, device=device, dtype=torch.float64) / a)).reshape(-1, 1)
            for p, a in zip(where, parts)]


def _plain_rotary(case, s):
    n, d = case["n"], case["head_dim"]
    turned = case["q_heads"] + case["kv_heads"]
    x = s["x"].float().reshape(n, -1, d, _cells(case["dims"]))
    sign = 1.0 if case["do"] == "forward" else -1.0
    out, first = [], 0
    for angle in _angles(case, x.device):
        half = angle.shape[0]
        a, b = x[:, :turned, first:first + half], x[:, :turned, first + half:first + 2 * half]
        cos, sin = angle.cos().float(), sign * angle.sin().float()
        out += [a * cos - b * sin, a * sin + b * cos]
        first += 2 * half
    out.append(x[:, :turned, first:])
    y = torch.cat([torch.cat(out, 2), x[:, turned:]], 1)
    return {"y": y.reshape(s["y"].shape).to(s["y"].dtype)}


def _heads(case, s, prefix=""):
    """q, k, v as [n, kv_heads, queries of a group or 1, head_dim, cells]."""
    n, d, h, g = case["n"], case["head_dim"], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    q_ch, kv_ch = case["q_heads"] * d, h * d
    if prefix + "qkv" in s:
        q, k, v = s[prefix + "qkv"].flatten(2).split([q_ch, kv_ch, kv_ch], 1)
    else:
        q, (k, v) = s[prefix + "q"].flatten(2), s[prefix + "kv"].flatten(2).split([kv_ch, kv_ch], 1)
    return q.reshape(n, h, g, d, -1), k.reshape(n, h, 1, d, -1), v.reshape(n, h, 1, d, -1)


def _allowed(case, s, device):
    """Which key a query may see, [n or 1, 1, 1, queries, keys], or None."""
    sq, sk = _cells(case["q_dims"]), _cells(case["kv_dims"])
    ok = None
    if case["causal"]:
        i, j = torch.arange(sq, device=device), torch.arange(sk, device=device)
        ok = (j[None, :] <= i[:, None] + (sk - sq))[None, None, None]
    if s["kv_mask"] is not None:
        m = s["kv_mask"][:, None, None, None, :]
        ok = m if ok is None else ok & m
    if s["q_mask"] is not None:
        ok = ok & s["q_mask"][:, None, None, :, None]
    return ok


def _plain_attention(case, s):
    t = s["o"].dtype
    q, k, v = (x.float() for x in _heads(case, s))
    scale = 1.0 / math.sqrt(case["head_dim"])
    score = torch.matmul(q.transpose(-1, -2), k) * scale
    ok = _allowed(case, s, q.device)
    if ok is not None:
        score = score.masked_fill(~ok, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(v, p.transpose(-1, -2))
    got = {"o": o.reshape(s["o"].shape).to(t), "lse": (top + total.log()).reshape(s["lse"].shape)}
    if case["do"] == "train":
        d_o = s["d_o"].float().reshape(o.shape)
        d_p = torch.matmul(d_o.transpose(-1, -2), v)
        d_v = torch.matmul(d_o, p).sum(2)
        d_s = p * (d_p - (p * d_p).sum(-1, keepdim=True)) * scale
        del d_p, p, score
        d_q, d_k = torch.matmul(k, d_s.transpose(-1, -2)), torch.matmul(q, d_s).sum(2)
        flat = [x.reshape(case["n"], -1, x.shape[-1]).to(t) for x in (d_q, d_k, d_v)]
        if "d_qkv" in s:
            got["d_qkv"] = torch.cat(flat, 1).reshape(s["qkv"].shape)
        else:
            got["d_q"], got["d_kv"] = flat[0].reshape(s["q"].shape), torch.cat(flat[1:], 1).reshape(s["kv"].shape)
    return got


def run(s):
    if own:
        return _run_own(s)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention}[s["case"]["op"]](s["case"], s)


def work(case):
    size = {"f32": 4, "bf16": 2}
    if case["op"] == "norm":
        cells, e = case["n"] * _cells(case["dims"]), size[case["dtype"]]
        # forward: x, y, two statistics a cell; backward: x, dy, dx, the statistics
        moved = cells * (2 * case["c"] * e + 8)
        flops = 8 * cells * case["c"]
        if case["do"] == "train":
            moved += cells * (3 * case["c"] * e + 8)
            flops += 14 * cells * case["c"]
        return {"bytes": moved, "flops": flops}
    if case["op"] == "rotary":
        values = case["n"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["head_dim"] * _cells(case["dims"])
        return {"bytes": values * (size[case["dtype"]] + size[case["to"]]), "flops": 3 * values}
    d, e = case["head_dim"], size[case["dtype"]]
    q_mask, kv_mask = _masks(case)
    sq, sk, n = _cells(case["q_dims"]), _cells(case["kv_dims"]), case["n"]
    keys = [sk] * n if kv_mask is None else kv_mask.sum(1).tolist()
    queries = [sq] * n if q_mask is None else q_mask.sum(1).tolist()
    pairs = case["q_heads"] * sum(a * b for a, b in zip(queries, keys))
    if case["causal"]:
        pairs *= 0.5
    q_side, kv_side = n * case["q_heads"] * sq, n * case["kv_heads"] * sk
    moved, flops = e * d * (2 * q_side + 2 * kv_side) + 4 * q_side, 4 * d * pairs
    if case["do"] == "train":
        # q, o, d_o, lse and k, v in; d_q, d_k, d_v out; five products
        moved += e * d * (4 * q_side + 4 * kv_side) + 4 * q_side
        flops += 10 * d * pairs
    return {"bytes": moved, "flops": flops}


# ---- their definition, in 64 bits ----------------------------------------------------------------------------------


def _exact_norm(case, s):
    leaf = s["x"].double().requires_grad_()
    w, b = s["scale"].double().requires_grad_(), s["bias"].double().requires_grad_()
    rows = leaf.movedim(1, -1)
    var, mean = torch.var_mean(rows, -1, correction=0)
    y = ((rows - mean[..., None]) / torch.sqrt(var + EPS)[..., None] * w + b).movedim(-1, 1)
    got = {"y": y.detach(), "mean": mean.detach().flatten(1), "inv_std": (1 / torch.sqrt(var + EPS)).detach().flatten(1)}
    if case["do"] == "train":
        got["d_x"], got["d_scale"], got["d_bias"] = torch.autograd.grad(y, (leaf, w, b), s["d_y"].double())
    return got


def _exact_rotary(case, s):
    n, d, cells = case["n"], case["head_dim"], _cells(case["dims"])
    y = s["x"].double().reshape(n, -1, d, cells).clone()
    ext = _ext(case["dims"])
    index = torch.arange(cells, device=y.device)
    at = {}
    for axis in range(len(ext) - 1, -1, -1):
        at[axis] = (index % ext[axis]).double()
        index = index // ext[axis]
    channel, turned = 0, case["q_heads"] + case["kv_heads"]
    for axis, a in enumerate(_axis_channels(d, len(ext))[3 - len(ext):]):
        for j in range(a // 2):
            angle = at[axis] * BASE ** (-2.0 * j / a)
            turn = torch.polar(torch.ones_like(angle), angle if case["do"] == "forward" else -angle)
            i0, i1 = channel + j, channel + a // 2 + j
            z = torch.complex(y[:, :turned, i0], y[:, :turned, i1]) * turn
            y[:, :turned, i0], y[:, :turned, i1] = z.real, z.imag
        channel += a
    return {"y": y.reshape(s["y"].shape)}


def _exact_attention(case, s):
    """One head after the other, its gradients by differentiation."""
    d, group, n = case["head_dim"], case["q_heads"] // case["kv_heads"], case["n"]
    q_ch, kv_ch = case["q_heads"] * d, case["kv_heads"] * d
    train = case["do"] == "train"
    packed = "qkv" in s
    src = [s["qkv"]] if packed else [s["q"], s["kv"]]
    flat = [x.flatten(2) for x in src]
    grads = [torch.zeros(x.shape, dtype=torch.float64, device=x.device) for x in flat]
    sq, sk = _cells(case["q_dims"]), _cells(case["kv_dims"])
    o = torch.zeros((n, q_ch, sq), dtype=torch.float64, device=flat[0].device)
    lse = torch.full((n, case["q_heads"], sq), -math.inf, dtype=torch.float64, device=o.device)
    k_at = q_ch if packed else 0
    for b in range(n):
        rows = torch.arange(sq, device=o.device) if s["q_mask"] is None else s["q_mask"][b].nonzero()[:, 0]
        cols = torch.arange(sk, device=o.device) if s["kv_mask"] is None else s["kv_mask"][b].nonzero()[:, 0]
        for h in range(case["q_heads"]):
            kv0 = k_at + h // group * d
            q = flat[0][b, h * d:(h + 1) * d].double()[:, rows].T.requires_grad_(train)
            k = flat[-1][b, kv0:kv0 + d].double()[:, cols].T.requires_grad_(train)
            v = flat[-1][b, kv0 + kv_ch:kv0 + kv_ch + d].double()[:, cols].T.requires_grad_(train)
            z = q @ k.T / math.sqrt(d)
            if case["causal"]:
                z = torch.where(cols[None, :] <= rows[:, None] + sk - sq, z, -math.inf)
            norm = torch.logsumexp(z, 1)
            r = torch.exp(z - norm[:, None]) @ v
            o[b, h * d:(h + 1) * d, rows], lse[b, h, rows] = r.detach().T, norm.detach()
            if train:
                up = s["d_o"].flatten(2)[b, h * d:(h + 1) * d].double()[:, rows].T
                gq, gk, gv = torch.autograd.grad(r, (q, k, v), up)
                grads[0][b, h * d:(h + 1) * d, rows] = gq.T
                grads[-1][b, kv0:kv0 + d, cols] += gk.T
                grads[-1][b, kv0 + kv_ch:kv0 + kv_ch + d, cols] += gv.T
            del z, r
    got = {"o": o.reshape(s["o"].shape), "lse": lse}
    if train:
        names = ["d_qkv"] if packed else ["d_q", "d_kv"]
        got.update({k: g.reshape(x.shape) for k, g, x in zip(names, grads, src)})
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention}[case["op"]](case, s)
