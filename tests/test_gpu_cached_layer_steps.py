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


def test_steps_do_not_wait_for_the_gpu():
    """Once its buffers stand a step makes no call that torch knows to wait for the stream, and results
    of steps queued behind each other are those of steps that are waited for."""
    _, mats = build()
    b = nq.Backend(0)
    queued, waited = (CachedLayer(b, mats, sequences=3, pages=24, page_tokens=16, head_dim=D) for _ in range(2))
    rng = np.random.default_rng(41)
    steps = [([30, 40, 10], to_gpu(rng.standard_normal((80, HIDDEN)).astype(np.float32)))]
    for _ in range(6):
        steps.append(([1, 1, 1], to_gpu(rng.standard_normal((3, HIDDEN)).astype(np.float32))))
        steps.append(([1, 0, 4], to_gpu(rng.standard_normal((5, HIDDEN)).astype(np.float32))))
    want = []
    for counts, x in steps:
        want.append(waited.forward(x, counts).clone())
        b.sync()
    got = [queued.forward(steps[0][1], steps[0][0]).clone()]
    b.sync()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got += [queued.forward(x, counts).clone() for counts, x in steps[1:]]
    finally:
        torch.cuda.set_sync_debug_mode("default")
    b.sync()
    for g, w in zip(got, want):
        assert bool((g == w).all())
    b.close()


def test_a_step_is_not_captured():
    """A graph would hold copies from host memory that another step has by then."""
    _, mats = build()
    b = nq.Backend(0)
    layer = CachedLayer(b, mats, sequences=1, pages=4, page_tokens=16, head_dim=D)
    x = to_gpu(np.random.default_rng(42).standard_normal((1, HIDDEN)).astype(np.float32))
    layer.forward(x, [1])
    b.sync()
    before = state_of(layer)
    other = torch.zeros(4, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        other += 1
        with pytest.raises(nq.InvalidArgument):
            layer.forward(x, [1])
    assert same(state_of(layer), before)
    graph.replay()
    layer.forward(x, [1])
    b.sync()
    assert layer.lengths == [2] and bool((other == 1).all())
    b.close()
