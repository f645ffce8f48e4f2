"""How much of a softmax's weights the attention keeps (nuq_cache_attention, include/nuq.h): one token
that dominates over many equal small ones, where roundings of equal weights add up instead of averaging out.

Bounds, derived from the arithmetic. Scores are single products here, exact but for the scale (two roundings,
2^-23 of at most 16 in powers of two) and one F32 fma of a magnitude below 32 (2^-20): 2^-18.4 in powers of two,
a relative 2^-18.9 of a weight, and 2^-22 for its exponential; the normaliser carries the same, so 2^-17 of the
weighted magnitudes in all. F32 sums run over steps of at least 16 tokens, four waves in turn: 2^-24 each for the
weights and the output. Weights are held to 2^-22 of themselves in two f16 parts, and below f16's normal range to
2^-25 where the row's largest is at least 2^7: 2^-32 of the row's sum each. F16 queries keep one part, 2^-11 of a
weight, and round the output."""
import numpy as np
import pytest

import nuclis_amd as nq
from oracle import cache_oracle as co
from tests.test_gpu_attention import Case, prompt_table

pytestmark = pytest.mark.gpu

# how far (in powers of two) the many lie below the one: weights that lie nearly half way between f16 numbers
LOGS = [e - np.log2(1 + (2 * k + 0.9) / 2048) for e, k in ((15, 1), (15, 40), (14, 3), (12, 9), (9, 2), (5, 30))]


@pytest.fixture(scope="module")
def backend():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return nq.Backend(0)


def bound_of(length, mass, plain, o, f16):
    bound = (2.0 ** -17 + 2.0 ** -23 * -(-length // 64)) * mass + 2.0 ** -32 * plain
    return bound + (2.0 ** -11 * mass + 2.0 ** -11 * np.abs(o) + 2.0 ** -25 if f16 else 0.0)


def one_over_many(backend, length, tokens, log, dtype, where):
    """Keys of zeros but for one token's first value, values of 1 but for its -1."""
    import torch
    c = Case([length], [tokens], kv=1, group=1, d=64, page=64, dtype=dtype, seed=1)
    k, v = np.zeros((length, 1, 64), np.float32), np.ones((length, 1, 64), np.float32)
    k[where, 0, 0], v[where, 0] = 8.0, -1.0
    c.write(backend, 0, k, v)
    torch.cuda.synchronize()
    c.q = np.zeros_like(c.q)
    c.q[:, 0, 0] = log * np.log(2)
    return c


def check(c, got, length, tokens, rows):
    f16 = c.dtype.itemsize == 2
    for i in rows:
        o, mass, plain, _ = co.attention(c.q[i:i + 1], *c.values[0], length - tokens + i, 1, 0.125)
        share = np.abs(got[i:i + 1] - o) / bound_of(length, mass, plain, o, f16)
        assert share.max() <= 1, (length, i, float(share.max()))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("length,bound", [(301, 0), (9001, 0), (9001, 1), (32768, 0)])
def test_one_token_over_many_equal_ones(backend, dtype, length, bound):
    """One workgroup (a bound of one token on the length) and many."""
    for i, log in enumerate(LOGS):
        c = one_over_many(backend, length, 1, log, dtype, (5, length // 2, length - 1)[i % 3])
        check(c, c.run(backend, scale=0.125, max_length=bound), length, 1, [0])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("length", [301, 4500])
def test_prompt_rows_over_many_equal_tokens(backend, dtype, length):
    for i, log in enumerate(LOGS):
        c = one_over_many(backend, length, 70, log, dtype, (5, length // 2, length - 60)[i % 3])
        check(c, c.run(backend, scale=0.125, table=prompt_table(c)), length, 70, [0, 1, 11, 50, 69])


@pytest.mark.parametrize("length", [301, 9001, 32768])
def test_one_part_of_the_weights_would_be_seen(length):
    """The F32 bound against weights of a single f16 part, in float64 on the host."""
    seen = []
    for log in LOGS:
        w = np.array([2.0 ** 7, 2.0 ** (7 - log)])
        held = w.astype(np.float16).astype(np.float64)
        count = np.array([1, length - 1])
        o, got = (count * w * [-1, 1]).sum() / (count * w).sum(), (count * held * [-1, 1]).sum() / (count * w).sum()
        seen.append(abs(got - o) / bound_of(length, 1.0, float(length), o, False))
    assert max(seen) > 2


@pytest.mark.parametrize("held,brought,kw", [([9001], [1], {}), ([9001], [1], dict(max_length=1)), ([5000, 32000], [2, 2], {})])
def test_long_axes_of_ordinary_rows(backend, held, brought, kw):
    """F32 rows as test_gpu_attention.py draws them, with this floor in place of 2^-24 of all values."""
    c = Case(held, brought, kv=1, group=5, seed=4)
    got = c.run(backend, **kw)
    at = 0
    for b, (n, new) in enumerate(zip(held, brought)):
        o, mass, plain, reach = co.attention(c.q[at:at + new], *c.values[b], n - new, 5, 128 ** -0.5)
        bound = (2 * 2.0 ** -20 * reach[..., None] + 2.0 ** -19) * mass + 2.0 ** -32 * plain
        assert np.all(np.abs(got[at:at + new] - o) <= bound), np.max(np.abs(got[at:at + new] - o) / bound)
        at += new
