"""The bounds that layer normalisation is tested with are tight enough to be broken: no GPU."""
import torch

import ln_ref


def test_a_lost_tile_or_zeros_break_the_bounds_of_the_parameter_gradients():
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(1, 8, 540000, generator=g) * s + m for s, m in ((2.0, 0.5), (1.0, 0.0)))
    want = ln_ref.layer_norm(x, None, None, 1e-5, dy, tiles_a_block=2)
    short = ln_ref.layer_norm(x[..., 128:], None, None, 1e-5, dy[..., 128:])  # without the first tile of a group
    for name in ("dscale", "dbias"):
        value, bound = want[name]
        assert bool((value.abs() > bound).any()) and bool(((value - short[name][0]).abs() > bound).any())
        assert int((value.abs() > bound).sum()) >= 7


def test_launches_are_dealt_out_as_documented():
    for (n, c, h, w), kind, more in (((1, 8, 1100, 1000), (4, 1, False), True), ((2, 64, 401, 301), (4, 8, True), True),
                                     ((900, 8, 15, 33), (1, 1, False), True), ((4, 16, 64, 64), (1, 4, False), False)):
        how = ln_ref.launch(c, h * w, n, 4 if h * w % 4 == 0 else 1, 148, True)
        assert (how["v"], how["g"], how["split"]) == kind and (how["tiles"] > how["blocks"]) == more
