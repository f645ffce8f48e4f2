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


def test_matrices_that_do_not_fit_each_other():
    """A v of more rows than k would be written past its place in the merged row; heads that are not whole
    have no place in the cache."""
    good = {"q": (384, 64), "k": (128, 64), "v": (128, 64), "o": (64, 384), "gate": (192, 64), "up": (192, 64),
            "down": (64, 192), "lm_head": (1000, 64)}
    changes = [{n: s} for n, s in (("v", (192, 64)), ("v", (64, 64)), ("k", (96, 64)), ("q", (320, 64)), ("o", (64, 320)),
                                   ("o", (128, 384)), ("up", (256, 64)), ("gate", (192, 32)), ("down", (64, 128)),
                                   ("lm_head", (1000, 128)))]
    changes += [{"k": (64, 64)}, {"k": (96, 64), "v": (96, 64)}, {"q": (320, 64), "o": (64, 320)}]
    for change in changes:
        mats = {n: SimpleNamespace(rows=r, columns=c) for n, (r, c) in {**good, **change}.items()}
        with pytest.raises(nq.InvalidShape):
            CachedLayer(SimpleNamespace(device="none"), mats, sequences=2, pages=4, head_dim=64)
