"""The cache oracle against the format's definition on the CPU, and the host's
size rules (no GPU)."""
import numpy as np
import pytest

import nuclis_amd as nq
from oracle import cache_oracle as co


def test_every_value_and_bias_is_an_f16_number():
    """What the kernels' single f16 fma rests on: d * code and bias * d are exact in f16 for every scale."""
    rng = np.random.default_rng(0)
    for bits, low, high, bias in ((4, -8, 7, 24), (8, -127, 127, 1152)):
        x = (rng.standard_normal((4000, 32)) * np.exp(rng.uniform(-18, 13, (4000, 1)))).astype(np.float32)
        _, d = co.quantise(bits, x)
        d = np.unique(d).astype(np.float64)
        for code in list(range(low, high + 1)) + [bias]:
            assert np.array_equal((d * code).astype(np.float16).astype(np.float64), d * code), (bits, code)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_layout_uses_every_bit_of_a_tile_once(bits, d):
    tile = co.geometry(bits, d)[3]
    used = np.zeros(tile * 8, int)
    scales = set()
    for place in (co.k_place, co.v_place):
        for t in range(16):
            for c in range(d):
                byte, bit, scale = place(bits, d, t, c)
                used[byte * 8 + bit:byte * 8 + bit + bits] += 1
                scales.add(scale)
    for s in scales:
        used[s * 8:s * 8 + 16] += 1
    assert np.all(used == 1)


def test_codes_by_hand():
    x = np.zeros(32, np.float32)
    x[:4] = [4.0, -4.0, 1.0, 0.26]
    q, d = co.quantise(4, x)                     # the positive one of the tie: d = -4 / 8
    assert d[0] == -0.5 and q[:4].tolist() == [-8, 7, -2, -1]
    q, d = co.quantise(8, x)                     # 4 / 127 = 0.0315 up to 4 bits: 0.03125 * 1.125
    assert d[0] == np.float16(0.03515625) and q[:3].tolist() == [114, -114, 28]


def test_cache_bytes():
    assert nq.cache_bytes(4, 10, 64, 8, 128) == 10 * 8 * 4 * 2304
    assert nq.cache_bytes(8, 1, 16, 1, 256) == 256 * 34
    for bad in ((5, 1, 16, 1, 64), (4, 0, 16, 1, 64), (4, 1, 24, 1, 64), (4, 1, 8, 1, 64), (4, 1, 16, 0, 64),
                (4, 1, 16, 1, 96), (4, 1, 8192, 1, 64), (4, 1 << 31, 16, 1, 64), (4, 1, 16, 1 << 20, 64),
                (-4, 1, 16, 1, 64)):
        with pytest.raises(nq.InvalidShape):
            nq.cache_bytes(*bad)


def test_attention_oracle_by_hand():
    """Two tokens of equal scores: the mean; a window of one: the last; nothing in reach: zeros."""
    k = np.zeros((2, 1, 64))
    v = np.stack([np.full((1, 64), 1.0), np.full((1, 64), 3.0)])
    q = np.ones((1, 2, 64), np.float32)
    o, mass, _, _ = co.attention(q, k, v, 1, 2, 1.0)
    assert np.allclose(o, 2.0) and np.allclose(mass, 2.0)
    assert np.allclose(co.attention(q, k, v, 1, 2, 1.0, window=1)[0], 3.0)
    assert not co.attention(q, k, v, -1, 2, 1.0)[0].any()
