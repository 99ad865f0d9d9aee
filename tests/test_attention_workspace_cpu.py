"""Workspace sizes that the Python class of attention keeps: no GPU."""
import torch

import dihydrogen_b200 as dc
from dihydrogen_b200 import _abi
from test_attention_cpu import tensor


def test_sizes_are_asked_for_once_a_geometry_and_device(monkeypatch):
    """How much a call needs goes by the device's SMs, too."""
    asked = []

    class Library:
        def dcb_attention_workspace_bytes(self, ad, qd, kd, backward):
            asked.append(backward)
            return len(asked)

    monkeypatch.setattr(_abi, "lib", Library)

    class Backend:
        stream = None

    layer, sizes = dc.Attention(Backend(), 4, 2), {}
    for cells in (3, 5):
        q = tensor([cells, 1, 8, 1])
        q.allocate("cpu")
        for device in (0, 1, 0, 1, 1):
            got = layer._desc(q, q, q.local_shape, q.local_shape, device)[1]
            assert sizes.setdefault((cells, device), got) == got
    assert len(asked) == 2 * 4 and len({tuple(s) for s in sizes.values()}) == 4
    for cells in range(1, 200):
        q = tensor([cells, 2, 8, 1])
        q.allocate("cpu")
        layer._desc(q, q, q.local_shape, q.local_shape, 0)
    assert len(layer._known) == layer.KNOWN
