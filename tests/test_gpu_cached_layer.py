"""Sequences through a layer over the quantised cache (nuclis_amd/cached_layer.py):
every stage against float64, from the stage before as the GPU gave it.

Bars: products of more than 3 rows are f16 tiles, 2e-3 of the largest value as for
the layer (test_gpu_layer.py); the cache holds exactly what its definition gives for the GPU's
k and v; the attention within its own bound (2^-18 of the weighted magnitudes at these
scores, see test_gpu_attention.py); log probabilities within 2e-5: two roundings
of numbers below 256 (2^-17 each) and F32 sums of a thousand terms."""
import numpy as np
import pytest

import nuclis_amd as nq
from nuclis_amd.cached_layer import CachedLayer
from nuclis_amd.synth import gaussian
from oracle import cache_oracle as co
from oracle import layer_oracle
from oracle import oracle as orc
from tests.gpu_util import to_gpu

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, D, FFN, VOCAB = 512, 6, 2, 128, 768, 1000
SHAPES = {"q": (nq.Q4_K, HEADS * D, HIDDEN), "k": (nq.Q4_K, KV * D, HIDDEN), "v": (nq.Q4_K, KV * D, HIDDEN),
          "o": (nq.Q4_K, HIDDEN, HEADS * D), "gate": (nq.Q4_K, FFN, HIDDEN), "up": (nq.Q4_K, FFN, HIDDEN),
          "down": (nq.Q4_K, HIDDEN, FFN), "lm_head": (nq.Q6_K, VOCAB, HIDDEN)}


def build(seed=30, std=0.06):
    weights = {n: nq.quantize(e, gaussian(seed + i, (r, c), std)) for i, (n, (e, r, c)) in enumerate(SHAPES.items())}
    mats = {n: nq.Matrix(SHAPES[n][0], w.shape[0], SHAPES[n][2], to_gpu(w)) for n, w in weights.items()}
    return weights, mats


def product(weights, name, x):
    enc, rows, columns = SHAPES[name]
    return np.stack([orc.matvec(enc, rows, columns, weights[name], row) for row in np.ascontiguousarray(x, np.float32)])


def close(got, want, share=2e-3):
    assert np.abs(got - want).max() <= share * np.abs(want).max()


@pytest.mark.parametrize("bits,page,window", [(4, 64, 0), (8, 16, 0), (4, 16, 24)])
def test_prompts_chunks_and_tokens(bits, page, window):
    import torch
    weights, mats = build()
    b = nq.Backend(0)
    layer = CachedLayer(b, mats, sequences=3, pages=24, page_tokens=page, bits=bits, head_dim=D, window=window)
    rng = np.random.default_rng(31)
    held = [[np.zeros((0, KV, D))] * 2 for _ in range(3)]
    # prompts, a sequence that begins later, chunks beside single tokens, one token each, one token alone
    for counts in ([33, 0, 70], [1, 9, 1], [1, 1, 1], [0, 0, 1], [17, 2, 0], [1, 1, 1]):
        rows = sum(counts)
        x = rng.standard_normal((rows, HIDDEN)).astype(np.float32)
        logits = layer.forward(to_gpu(x), counts)
        targets = rng.integers(0, VOCAB, rows).astype(np.int32)
        scored = layer.score(logits, to_gpu(targets), top=4)
        b.sync()
        buffers = {n: t[:rows].cpu().numpy() for n, t in layer.buffers.items()}
        q, k, v = np.split(buffers["qkv"], [HEADS * D, (HEADS + KV) * D], 1)
        for name, got in (("q", q), ("k", k), ("v", v)):
            close(got, product(weights, name, x))
        at = 0
        for s, count in enumerate(counts):
            if count == 0:
                continue
            mine = slice(at, at + count)
            new = co.stored(bits, k[mine].reshape(-1, KV, D), v[mine].reshape(-1, KV, D))[:2]
            held[s] = [np.concatenate([old, n]) for old, n in zip(held[s], new)]
            assert len(held[s][0]) == layer.lengths[s]
            for i in range(at, at + count):
                o, mass, plain, reach = co.attention(q[i:i + 1].reshape(1, HEADS, D), *held[s],
                                                     layer.lengths[s] - count + i - at, HEADS // KV, D ** -0.5, window)
                bound = (2 * 2.0 ** -20 * reach[..., None] + 2.0 ** -19) * mass + 2.0 ** -24 * plain
                assert np.all(np.abs(buffers["attn"][i].reshape(1, HEADS, D) - o) <= bound)
            at += count
        h1 = x + product(weights, "o", buffers["attn"])
        close(buffers["h1"], h1)
        act = layer_oracle.silu(product(weights, "gate", buffers["h1"])) * product(weights, "up", buffers["h1"])
        close(buffers["act"], act, 4e-3)  # of two products
        h2 = buffers["h1"] + product(weights, "down", buffers["act"])
        close(buffers["h2"], h2)
        got = logits.cpu().numpy()
        close(got, product(weights, "lm_head", buffers["h2"]))
        wide = got.astype(np.float64)
        assert np.ptp(wide, axis=1).max() < 256
        p = wide - wide.max(1, keepdims=True)
        p -= np.log(np.exp(p).sum(1, keepdims=True))
        assert np.abs(scored["logprobs"].cpu().numpy() - p[np.arange(rows), targets]).max() <= 2e-5
        assert np.abs(scored["entropy"].cpu().numpy() + (np.exp(p) * p).sum(1)).max() <= 2e-5
        order = np.argsort(-wide, axis=1, kind="stable")[:, :4]
        assert np.array_equal(scored["top_ids"].cpu().numpy(), order)
        assert np.abs(scored["top_logprobs"].cpu().numpy() - np.take_along_axis(p, order, 1)).max() <= 2e-5
    # what a step wrote is what the cache holds
    s = 0
    slots = layer.table[s, np.arange(layer.lengths[s]) // page].astype(np.int64) * page + np.arange(layer.lengths[s]) % page
    kr, vr = (torch.zeros(layer.lengths[s], KV, D, device="cuda") for _ in range(2))
    b.cache_read(layer.cache, to_gpu(slots), kr, vr)
    b.sync()
    assert np.array_equal(kr.cpu().numpy(), held[s][0]) and np.array_equal(vr.cpu().numpy(), held[s][1])
    b.close()


def test_pages_come_back_and_run_out():
    _, mats = build()
    b = nq.Backend(0)
    layer = CachedLayer(b, mats, sequences=2, pages=4, page_tokens=16, head_dim=D)
    rng = np.random.default_rng(32)
    x = to_gpu(rng.standard_normal((40, HIDDEN)).astype(np.float32))
    first = layer.forward(x, [40, 0]).clone()
    with pytest.raises(nq.InvalidShape):
        layer.forward(x, [0, 40])  # 3 pages, one is left
    assert layer.lengths == [40, 0]
    with pytest.raises(nq.InvalidShape):
        layer.forward(x, [40])
    layer.release(0)
    second = layer.forward(x, [0, 40])
    b.sync()
    assert bool((first == second).all())  # the same prompt on other pages
    assert layer.forward(x[:0], [0, 0]).shape == (0, VOCAB)
    b.close()
