"""What CachedLayer (nuclis_amd/cached_layer.py) refuses before it runs anything. No GPU is used:
tensors without memory stand for those on it."""
from types import SimpleNamespace

import pytest
import torch

import nuclis_amd as nq
from nuclis_amd.cached_layer import CachedLayer
from tests.test_cache_arguments import OnGpu


@pytest.fixture
def layer(monkeypatch):
    one = object.__new__(CachedLayer)
    one._torch, one.backend, one.hidden = torch, SimpleNamespace(device=0), 64
    one.lengths, one.pages = [0, 0], [[], []]
    one.ran = []
    monkeypatch.setattr(one, "_grow", lambda counts: one.ran.append(counts))
    monkeypatch.setattr(one, "_shrink", lambda before: None)
    monkeypatch.setattr(one, "_device", lambda array: array)
    if hasattr(one, "_step"):
        monkeypatch.setattr(one, "_step", lambda *args: None)
    return one


@pytest.mark.parametrize("rows", [1, 3])
def test_inputs(layer, rows):
    counts = [rows, 0]
    turned = OnGpu(rows, 64)
    turned._t = torch.empty(64, rows + 1, device="meta").t()[:rows]
    for x, error in ((OnGpu(rows, 64, dtype=torch.float16), nq.InvalidArgument),
                     (OnGpu(rows, 64, dtype=torch.float64), nq.InvalidArgument),
                     (torch.zeros(rows, 64), nq.InvalidArgument), (OnGpu(rows, 64, device=1), nq.InvalidArgument),
                     (OnGpu(rows, 63), nq.InvalidShape), (turned, nq.InvalidShape)):
        with pytest.raises(error):
            layer.forward(x, counts)
    assert layer.ran == [] and layer.lengths == [0, 0]
    layer.forward(OnGpu(rows, 64), counts)
    assert layer.ran == [counts]
