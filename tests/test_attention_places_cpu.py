"""Which results of attention may lie where: no GPU.  Every call is refused, for its workspace where its places are fine."""
import itertools
import random

import pytest

from dihydrogen_b200 import _abi
from test_attention_cpu import FAKE, desc, nd, status

FAR = 1 << 32


def packed(n, c, cells, of):
    """Descriptor of c channels of a tensor of `of` channels."""
    d = nd(n, c, 1, cells)
    d.sn = of * cells
    return d


def fwd(qd, kd, at, od=None):
    a = {k: FAKE + (i + 1) * FAR for i, k in enumerate(("q", "k", "v", "o", "lse", "qm", "km"))}
    a.update(at)
    st = status("dcb_attention_fwd", desc(q=2, kv=1, dtype=_abi.BF16), qd, a["q"], kd, a["k"], kd, a["v"], a["qm"], a["km"],
                od or qd, a["o"], a["lse"], None, 0, None)
    assert st == _abi.BAD_ARG
    return b"place" in _abi.lib().dcb_last_error()


def bwd(qd, kd, at, dqd=None, dkd=None):
    names = ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "qm", "km")
    a = {k: FAKE + (i + 1) * FAR for i, k in enumerate(names)}
    a.update(at)
    dkd = dkd or kd
    st = status("dcb_attention_bwd", desc(q=2, kv=1, dtype=_abi.BF16), qd, a["q"], kd, a["k"], kd, a["v"], a["qm"], a["km"],
                qd, a["o"], a["lse"], qd, a["d_o"], dqd or qd, a["dq"], dkd, a["dk"], dkd, a["dv"], None, 0, None)
    assert st == _abi.BAD_ARG
    return b"place" in _abi.lib().dcb_last_error()


def test_results_that_reach_into_an_operand():
    qd, kd = nd(2, 16, 3, 5), nd(2, 8, 3, 5)
    size = {"q": 2 * 16 * 15 * 2, "k": 2 * 8 * 15 * 2, "v": 2 * 8 * 15 * 2, "lse": 2 * 2 * 15 * 4, "qm": 30, "km": 30}
    size.update({"o": size["q"], "d_o": size["q"], "dq": size["q"], "dk": size["k"], "dv": size["k"]})
    assert not fwd(qd, kd, {}) and not bwd(qd, kd, {})
    for call, results, names in ((fwd, ("o", "lse"), ("q", "k", "v", "qm", "km", "o", "lse")),
                                 (bwd, ("dq", "dk", "dv"), tuple(size))):
        for r, x in itertools.product(results, names):
            if r == x:
                continue
            base = FAKE + 40 * FAR
            unit = 4 if "lse" in (r, x) else 2
            for off, shared in ((0, True), (size[x], False), (size[x] - unit, True), (-size[r], False),
                                (unit - size[r], True)):
                assert call(qd, kd, {x: base, r: base + off}) == shared, (r, x, off)


def test_slices_of_a_packed_gradient():
    """dq, dk and dv are channels of one tensor, whose samples lie apart; a channel too early is refused."""
    n, cells, of = 3, 20, 16 + 8 + 8
    qd, kd = packed(n, 16, cells, of), packed(n, 8, cells, of)
    row = cells * 2
    base = FAKE + 40 * FAR
    good = {"dq": base, "dk": base + 16 * row, "dv": base + 24 * row}
    assert not bwd(qd, kd, good)
    for name in ("dk", "dv"):
        assert bwd(qd, kd, {**good, name: good[name] - 2})
        assert bwd(qd, kd, {**good, name: good[name] - row})
    assert bwd(qd, kd, {**good, "dv": good["dv"] + 2})  # over the next sample's queries
    # every second channel, the others a gradient's
    for d in (qd, kd):
        d.sc, d.sn = 2 * cells, 64 * cells
    assert not fwd(qd, kd, {"q": base, "o": base + row}) and fwd(qd, kd, {"q": base, "o": base + row - 2})


def test_places_against_a_count_of_bytes():
    """Layouts of equal and of other strides at random: refused whenever they share a byte, and with equal strides only then."""
    rng = random.Random(5)
    seen = [0, 0]
    for _ in range(3000):
        n, cells = rng.randint(1, 3), rng.randint(1, 4)
        a, b = nd(n, 16, 1, cells), nd(n, 8, 1, cells)
        equal = rng.random() < 0.8
        strides = None
        for d in (a, b):
            if strides is None or not equal:
                sc = cells + rng.randint(0, cells)
                strides = (sc, rng.choice((17, 20, 32)) * sc) if rng.random() < 0.8 else (3 * cells + rng.randint(0, 3), cells)
            d.sc, d.sn = strides
        base = FAKE + 40 * FAR
        off = 2 * rng.randint(-40 * cells * n, 40 * cells * n)
        byte = lambda d, at: {at + 2 * (i * d.sn + j * d.sc + k) for i in range(d.n) for j in range(d.c) for k in range(cells)}
        shared = bool(byte(a, base) & byte(b, base + off))
        got = bwd(nd(n, 16, 1, cells), nd(n, 8, 1, cells), {"dq": base, "dk": base + off}, dqd=a, dkd=b)
        assert got or not shared
        if equal:
            assert got == shared
            seen[shared] += 1
    assert min(seen) > 200
