"""Steps of sequences through a layer over the quantised cache (nuclis_amd/cached_layer.py)
that fail, and how steps follow each other."""
import numpy as np
import pytest
import torch

import nuclis_amd as nq
from nuclis_amd.cached_layer import CachedLayer
from tests.gpu_util import to_gpu
from tests.test_gpu_cached_layer import D, HIDDEN, build

pytestmark = pytest.mark.gpu


def state_of(layer):
    return list(layer.lengths), [list(p) for p in layer.pages], list(layer.free), layer.table.copy()


def same(a, b):
    return a[:3] == b[:3] and np.array_equal(a[3], b[3])


@pytest.mark.parametrize("fails", ["cache_write", "cache_attention", "matmul", "_buffer"])
def test_a_step_that_fails_can_be_tried_again(monkeypatch, fails):
    """The sequences hold what they held, whatever call failed, and the step's results are those of a layer
    on which nothing did."""
    _, mats = build()
    rng = np.random.default_rng(40)
    steps = [([20, 0, 33], rng.standard_normal((53, HIDDEN)).astype(np.float32)),
             ([17, 5, 1], rng.standard_normal((23, HIDDEN)).astype(np.float32)),
             ([1, 1, 1], rng.standard_normal((3, HIDDEN)).astype(np.float32))]
    b = nq.Backend(0)
    plain, tried = (CachedLayer(b, mats, sequences=3, pages=12, page_tokens=16, head_dim=D) for _ in range(2))
    for i, (counts, x) in enumerate(steps):
        want = plain.forward(to_gpu(x), counts).clone()
        before = state_of(tried)
        if i:
            def refuse(*args, **more):
                raise nq.InvalidShape("InvalidShape: not now")
            with monkeypatch.context() as m:
                m.setattr(tried if fails == "_buffer" else b, fails, refuse)
                with pytest.raises(nq.InvalidShape):
                    tried.forward(to_gpu(x), counts)
            assert same(state_of(tried), before)
        got = tried.forward(to_gpu(x), counts)
        b.sync()
        assert bool((got == want).all())
        assert same(state_of(tried), state_of(plain))
    b.close()
