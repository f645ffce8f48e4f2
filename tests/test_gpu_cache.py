"""The quantised K/V cache on cuda:0 against oracle/cache_oracle.py: what a
write stores (bit for bit), what a read gives (exact), and refusals.

Bars: the stored value is the definition's, so reads equal the oracle's values
exactly, in F32 and F16; each value is within half a step of its input (plus the
half step by which a scale rounded to 8 bits can cut the largest one)."""
import numpy as np
import pytest

import nuclis_amd as nq
from oracle import cache_oracle as co
from tests.gpu_util import to_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return nq.Backend(0)


def values(seed, shape):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal(shape).astype(np.float32)
    x *= np.exp(rng.standard_normal(shape[:-1] + (1,))).astype(np.float32)
    return x


def slots_of(seed, count, capacity):
    return np.random.default_rng(seed).permutation(capacity)[:count].astype(np.int64)


GEOMETRIES = [(b, d, page, heads) for b in (4, 8) for d, page, heads in ((64, 16, 3), (128, 64, 8), (256, 32, 1))]


@pytest.mark.parametrize("bits,d,page,heads", GEOMETRIES)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("tokens", [1, 7, 129])
def test_round_trip_is_the_definitions(backend, bits, d, page, heads, dtype, tokens):
    import torch
    print(f"[cache] {bits} bits d {d} page {page} heads {heads} {dtype} tokens {tokens}", flush=True)
    pages = -(-tokens // page) + 2
    cache = nq.KVCache(bits, pages, page, heads, d)
    k, v = values(tokens + d, (tokens, heads, d)), values(tokens + d + 1, (tokens, heads, d))
    if dtype == "f16":
        k, v = k.astype(np.float16), v.astype(np.float16)
    # edges: all zeros, equal extremes of both signs, one value alone, tiny ones, large ones
    k[0, 0, :32] = 0
    k[0, 0, 32:64] = np.where(np.arange(32) % 2, 1.5, -1.5)
    v[0, 0, :32] = np.where(np.arange(32) == 5, -3.25, 0)
    v[0, 0, 32:64] = values(3, (32,)) * 1e-6
    k[-1, -1, :32] = np.linspace(-60000, 60000, 32)
    v[-1, -1, 32:64] = np.where(np.arange(32) == 0, 7e4 if dtype == "f32" else 6.5e4, 1)
    slots = slots_of(5, tokens, pages * page)
    backend.cache_write(cache, to_gpu(k), to_gpu(v), to_gpu(slots))
    want_k, want_v, _ = co.stored(bits, k.astype(np.float32), v.astype(np.float32))
    for out in (torch.float32, torch.float16):
        kr, vr = (torch.full((tokens, heads, d), 9.0, dtype=out, device="cuda") for _ in range(2))
        backend.cache_read(cache, to_gpu(slots), kr, vr)
        backend.sync()
        assert np.array_equal(kr.cpu().numpy().astype(np.float64), want_k)
        assert np.array_equal(vr.cpu().numpy().astype(np.float64), want_v)
    # within half a step of the input, but where the largest code is cut: at 4
    # bits by the scale's rounding (at most 2^-8 of 8 steps) or its missing +8
    q, scale = co.quantise(bits, k.astype(np.float32))
    step = np.abs(scale.astype(np.float64)).repeat(32, -1)
    fine = np.abs(k.astype(np.float64)) < 5000
    bound = step * (0.5 + (1.0 if bits == 4 else 1e-6)) + 2.0 ** -24
    assert np.all(np.abs(want_k - k.astype(np.float64))[fine] <= bound[fine])


@pytest.mark.parametrize("bits,d,page,heads", GEOMETRIES)
def test_bytes_are_laid_out_as_documented(backend, bits, d, page, heads):
    """Every code and scale of two tiles by the layout's formulas."""
    tokens = 32
    pages = 3
    cache = nq.KVCache(bits, pages, page, heads, d)
    k, v = values(40, (tokens, heads, d)), values(41, (tokens, heads, d))
    first = page  # the second page's start
    backend.cache_write(cache, to_gpu(k), to_gpu(v), to_gpu(np.arange(first, first + tokens)))
    backend.sync()
    tile_bytes = co.geometry(bits, d)[3]
    raw = cache.bytes.cpu().numpy().reshape(pages, heads, page // 16, tile_bytes)
    want_k, want_v, _ = co.stored(bits, k, v)
    for head in range(heads):
        for t in range(tokens // 16):
            slot = first + 16 * t
            tile = raw[slot // page, head, slot % page // 16]
            assert np.array_equal(co.tile_values(bits, d, tile, co.k_place), want_k[16 * t:16 * t + 16, head])
            assert np.array_equal(co.tile_values(bits, d, tile, co.v_place), want_v[16 * t:16 * t + 16, head])
    assert not raw[0].any()  # the other pages are untouched


@pytest.mark.parametrize("bits,d", [(4, 64), (4, 128), (8, 128), (4, 256), (8, 256)])
def test_non_finite_values_poison_their_token_and_head(backend, bits, d):
    import torch
    tokens, heads, page = 9, 2, 16
    cache = nq.KVCache(bits, 1, page, heads, d)
    k, v = values(7, (tokens, heads, d)), values(8, (tokens, heads, d))
    k[1, 0, d - 1] = np.nan
    v[3, 1, 0] = np.inf
    k[4, 0, 17] = -np.inf
    v[8, 1, d // 2] = np.nan
    backend.cache_write(cache, to_gpu(k), to_gpu(v), torch.arange(tokens, device="cuda"))
    kr, vr = (torch.zeros(tokens, heads, d, device="cuda") for _ in range(2))
    backend.cache_read(cache, torch.arange(tokens, device="cuda"), kr, vr)
    backend.sync()
    want_k, want_v, bad = co.stored(bits, k, v)
    assert bad.sum() == 4
    assert np.array_equal(kr.cpu().numpy().astype(np.float64), want_k, equal_nan=True)
    assert np.array_equal(vr.cpu().numpy().astype(np.float64), want_v, equal_nan=True)


def test_strided_inputs_padding_slots_and_untouched_neighbours(backend):
    """K and V as slices of a merged q/k/v projection; -1 and out-of-range
    slots skip their tokens and read as zeros; other tokens keep their bytes."""
    import torch
    bits, d, heads, page, pages, tokens = 4, 128, 8, 32, 4, 50
    cache = nq.KVCache(bits, pages, page, heads, d)
    old_k, old_v = values(20, (pages * page, heads, d)), values(21, (pages * page, heads, d))
    everything = torch.arange(pages * page, device="cuda")
    backend.cache_write(cache, to_gpu(old_k), to_gpu(old_v), everything)
    merged = to_gpu(values(22, (tokens, 48 + 16, d)))
    k, v = merged[:, 48:56], merged[:, 56:64]
    slots = slots_of(23, tokens, pages * page)
    slots[[0, 10, 49]] = [-1, pages * page, -(1 << 40)]
    backend.cache_write(cache, k, v, to_gpu(slots))
    kr, vr = (torch.zeros(pages * page, heads, d, device="cuda") for _ in range(2))
    backend.cache_read(cache, everything, kr, vr)
    want_k, want_v, _ = co.stored(bits, old_k, old_v)
    new_k, new_v, _ = co.stored(bits, k.cpu().numpy(), v.cpu().numpy())
    live = (slots >= 0) & (slots < pages * page)
    want_k[slots[live]], want_v[slots[live]] = new_k[live], new_v[live]
    backend.sync()
    assert np.array_equal(kr.cpu().numpy().astype(np.float64), want_k)
    assert np.array_equal(vr.cpu().numpy().astype(np.float64), want_v)
    wide = torch.full((tokens, heads + 3, d), 5.0, device="cuda")  # strided outputs
    vw = torch.full((tokens, heads, d), 5.0, device="cuda")
    backend.cache_read(cache, to_gpu(slots), wide[:, :heads], vw)
    backend.sync()
    assert not wide[0, :heads].any() and not vw[10].any() and not vw[49].any()
    assert bool((wide[:, heads:] == 5.0).all())
    assert np.array_equal(wide[1:10, :heads].cpu().numpy().astype(np.float64), new_k[1:10])


def test_offsets_past_32_bits(backend):
    """Pages behind the first 4 GiB of a long cache."""
    import torch
    bits, d, heads, page = 4, 128, 8, 64
    pages = (5 << 30) // nq.cache_bytes(bits, 1, page, heads, d)
    cache = nq.KVCache(bits, pages, page, heads, d)
    tokens = 70
    k, v = values(30, (tokens, heads, d)), values(31, (tokens, heads, d))
    slots = np.concatenate([np.arange(35), pages * page - 1 - np.arange(35)]).astype(np.int64)
    backend.cache_write(cache, to_gpu(k), to_gpu(v), to_gpu(slots))
    kr, vr = (torch.zeros(tokens, heads, d, device="cuda") for _ in range(2))
    backend.cache_read(cache, to_gpu(slots), kr, vr)
    backend.sync()
    want_k, want_v, _ = co.stored(bits, k, v)
    assert np.array_equal(kr.cpu().numpy().astype(np.float64), want_k)
    assert np.array_equal(vr.cpu().numpy().astype(np.float64), want_v)


def test_refusals_leave_the_cache_untouched(backend):
    import torch
    cache = nq.KVCache(4, 2, 16, 2, 64)
    k = torch.ones(3, 2, 64, device="cuda")
    slots = torch.arange(3, device="cuda")
    shifted = torch.ones(3 * 2 * 64 + 1, device="cuda")[1:].view(3, 2, 64)
    for bad_k, bad_v, bad_slots, error in (
            (k[:2], k, slots, nq.InvalidShape), (k, k.half(), slots, nq.InvalidArgument),
            (k.double(), k.double(), slots, nq.InvalidArgument), (k, k, slots.int(), nq.InvalidArgument),
            (shifted, k, slots, nq.InvalidShape), (k, k[..., ::2].repeat(1, 1, 2)[:, :, :32], slots, nq.InvalidShape),
            (k.transpose(1, 2).contiguous().transpose(1, 2), k, slots, nq.InvalidShape),
            (torch.ones(3, 128 + 1, device="cuda")[:, :128].view(3, 2, 64), k, slots, nq.InvalidShape),
            (k, k, torch.arange(6, device="cuda")[::2], nq.InvalidShape)):
        with pytest.raises(error):
            backend.cache_write(cache, bad_k, bad_v, bad_slots)
        with pytest.raises(error):
            backend.cache_read(cache, bad_slots, bad_k, bad_v)
    with pytest.raises(nq.InvalidByteLength):
        backend.cache_write(nq.KVCache(4, 3, 16, 2, 64, cache.bytes), k, k, slots)
    misplaced = torch.zeros(cache.bytes.numel() + 8, dtype=torch.uint8, device="cuda")[8:]
    with pytest.raises(nq.InvalidShape):
        backend.cache_write(nq.KVCache(4, 2, 16, 2, 64, misplaced), k, k, slots)
    backend.sync()
    assert not cache.bytes.any() and not misplaced.any()
    none = torch.empty(0, 2, 64, device="cuda")
    backend.cache_write(cache, none, none, slots[:0])  # no tokens: nothing to do


def test_writes_and_reads_replay_from_a_graph_on_another_stream(backend):
    """Captured on a side stream, replayed with new inputs and eager work between."""
    import torch
    bits, d, heads, page = 4, 128, 8, 64
    cache = nq.KVCache(bits, 2, page, heads, d)
    k, v = torch.zeros(5, heads, d, device="cuda"), torch.zeros(5, heads, d, device="cuda")
    kr, vr = torch.zeros_like(k), torch.zeros_like(v)
    slots = torch.tensor([3, 64, 65, 127, 0], device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        backend.cache_write(cache, k, v, slots)
        backend.cache_read(cache, slots, kr, vr)
    for replay in range(3):
        a, b = values(60 + replay, (5, heads, d)), values(70 + replay, (5, heads, d))
        k.copy_(to_gpu(a)), v.copy_(to_gpu(b))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want_k, want_v, _ = co.stored(bits, a, b)
        assert np.array_equal(kr.cpu().numpy().astype(np.float64), want_k)
        assert np.array_equal(vr.cpu().numpy().astype(np.float64), want_v)


@pytest.mark.parametrize("bits", [4, 8])
def test_codes_at_the_edges_between_them(backend, bits):
    """Inputs at (c + 1/2) d and one F32 step to either side of it, for every code and for
    scales from the smallest an f16 holds to the largest kept: the codes are those of
    IEEE's quotient, rounded to even."""
    import torch
    top, steps = (8, 8) if bits == 4 else (127, 4)
    rng = np.random.default_rng(50)
    mantissas = 1 + rng.integers(0, 1 << (steps - 1), 40) / (1 << (steps - 1))
    scales = (mantissas * 2.0 ** rng.integers(-24, 11 if bits == 4 else 5, 40)).astype(np.float16).astype(np.float32)
    groups = []
    for d in scales:
        middles = ((np.arange(-top, top) + 0.5) * np.float64(d)).astype(np.float32)
        around = np.concatenate([np.nextafter(middles, np.float32(-np.inf)), middles, np.nextafter(middles, np.float32(np.inf))])
        around = np.resize(around, -(-len(around) // 31) * 31).reshape(-1, 31)
        # the extreme that makes the group's scale d
        groups.append(np.concatenate([around, np.full((len(around), 1), -top * d if bits == 4 else top * d, np.float32)], 1))
    x = np.concatenate(groups)
    x = np.resize(x, (-(-len(x) // 4) * 4, 32)).reshape(-1, 1, 128)
    cache = nq.KVCache(bits, -(-len(x) // 64), 64, 1, 128)
    slots = torch.arange(len(x), device="cuda")
    backend.cache_write(cache, to_gpu(x), to_gpu(-x), slots)
    kr, vr = (torch.zeros(len(x), 1, 128, device="cuda") for _ in range(2))
    backend.cache_read(cache, slots, kr, vr)
    backend.sync()
    want_k, want_v, _ = co.stored(bits, x, -x)
    assert np.array_equal(kr.cpu().numpy().astype(np.float64), want_k)
    assert np.array_equal(vr.cpu().numpy().astype(np.float64), want_v)


@pytest.mark.parametrize("bits", [4, 8])
def test_the_largest_numbers_of_f32(backend, bits):
    import torch
    x = values(51, (40, 2, 64))
    x[::3, 0] *= np.float32(3e37)
    x[1, 1, ::5] = np.finfo(np.float32).max
    x[2, 1, ::7] = -np.finfo(np.float32).max
    x[5, 0] = np.float32(1e-40)
    cache = nq.KVCache(bits, 3, 16, 2, 64)
    slots = torch.arange(40, device="cuda")
    backend.cache_write(cache, to_gpu(x), to_gpu(-x), slots)
    kr, vr = (torch.zeros(40, 2, 64, device="cuda") for _ in range(2))
    backend.cache_read(cache, slots, kr, vr)
    backend.sync()
    want_k, want_v, _ = co.stored(bits, x, -x)
    assert np.array_equal(kr.cpu().numpy().astype(np.float64), want_k)
    assert np.array_equal(vr.cpu().numpy().astype(np.float64), want_v)
