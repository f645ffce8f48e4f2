"""Calls of the attention over the quantised cache whose bounds are not the batch's own
counts (nuq_cache_attention, include/nuq.h), against the float64 oracle under the
bounds of test_gpu_attention.py."""
import numpy as np
import pytest

import nuclis_amd as nq
from tests.gpu_util import to_gpu
from tests.test_gpu_attention import Case, prompt_table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return nq.Backend(0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [0, 21])
def test_rows_before_a_bound_keep_their_positions(backend, dtype, window):
    """Sequences of more new tokens than max_tokens: the rows before it see what they see without
    the bound, the others stay as they are."""
    c = Case([40, 50, 3], [4, 4, 4], kv=1, group=2, d=64, page=16, dtype=dtype, seed=8)
    c.check(c.run(backend, window=window), window=window)
    got = c.run(backend, starts=np.array([0, 4, 8, 12]), max_tokens=2, window=window)
    c.check(got, window=window, rows=np.arange(2))
    for b in range(3):
        assert np.all(got[4 * b + 2:4 * b + 4] == 7.0)
    assert not got[8:9].any()  # the third one's first token stands before its start


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [0, 45])
def test_prompt_rows_before_a_bound_keep_their_positions(backend, dtype, window):
    c = Case([531, 90], [70, 80], kv=1, group=3, page=16, dtype=dtype, seed=26)
    got = c.run(backend, starts=np.array([0, 70, 150]), max_tokens=66, table=prompt_table(c), window=window)
    c.check(got, window=window, rows=np.arange(66))
    assert np.all(got[66:70] == 7.0) and np.all(got[136:] == 7.0)


@pytest.mark.parametrize("prompt", [False, True])
def test_rows_before_the_end_of_the_queries_keep_their_positions(backend, prompt):
    """Starts that name more rows than there are."""
    c = Case([300, 120], [30, 40], kv=1, group=3, page=16, seed=27)
    q = to_gpu(c.q)[:55].contiguous()
    got = c.run(backend, q=q, starts=np.array([0, 30, 70]), max_tokens=40,
                **(dict(table=prompt_table(c)) if prompt else {}))
    c.check(np.concatenate([got, np.zeros((15, 3, 128))]), rows=np.arange(25))
    # a count past any the sequence can hold: every row stands before its start
    got = c.run(backend, q=q, starts=np.array([0, 30, 2**31 - 1]), max_tokens=40)
    assert not got[30:].any()


def in_long_context(c, tokens):
    """The case's page table with entries for so many tokens, as one sized for a model's longest context."""
    table = np.full((len(c.held), max(tokens // c.page, c.table.shape[1])), -1, np.int32)
    table[:, :c.table.shape[1]] = c.table
    return table


@pytest.mark.parametrize("heads,tokens,batch,context", [(32, 2048, 256, 16384), (64, 2048, 128, 8192), (48, 1000, 400, 16384)])
def test_a_chunk_among_many_single_tokens_of_long_contexts(backend, heads, tokens, batch, context):
    """Both plans of the call split their axes."""
    print(f"[attention] chunk of {tokens} among {batch} sequences, {heads} heads, context {context}", flush=True)
    rng = np.random.default_rng(28)
    held = [tokens + 70] + [int(n) for n in rng.integers(1, 40, batch - 1)]
    c = Case(held, [tokens] + [1] * (batch - 1), kv=8, group=heads // 8, dtype="f16", seed=29)
    got = c.run(backend, table=in_long_context(c, context), max_tokens=tokens, max_length=context)
    c.check(got, rows=[0, 1, 63, 64, 500, tokens - 2, tokens - 1])


@pytest.mark.parametrize("dtype,heads,batch,context", [("f16", 64, 512, 8192), ("f32", 48, 600, 4096)])
def test_single_tokens_with_starts_and_no_bound(backend, dtype, heads, batch, context):
    print(f"[attention] {batch} single tokens with starts, {heads} heads, context {context} {dtype}", flush=True)
    held = [int(n) for n in np.random.default_rng(30).integers(0, 30, batch)]
    held[7] = 900
    c = Case(held, [1] * batch, kv=8, group=heads // 8, dtype=dtype, seed=31)
    c.check(c.run(backend, table=in_long_context(c, context), starts=np.arange(batch + 1)))


def test_rows_that_are_not_whole_sequences_are_refused(backend):
    """Without starts every sequence brings the same count: fewer rows than sequences, a count of none, or no
    sequences at all leave rows over."""
    import torch
    c = Case([20, 20, 20, 20], [1] * 4, kv=1, group=2, d=64, page=16, seed=32)
    q, table, lengths = to_gpu(c.q), to_gpu(c.table), to_gpu(np.array(c.held, np.int32))
    out = torch.full(q.shape, 7.0, device="cuda")
    for rows, batch, more in ((3, 4, {}), (4, 4, dict(max_tokens=0)), (4, 0, {}), (2, 0, dict(max_tokens=1))):
        with pytest.raises(nq.InvalidShape):
            backend.cache_attention(c.cache, q[:rows], out[:rows], table[:batch], lengths[:batch], **more)
    backend.sync()
    assert bool((out == 7.0).all())
    backend.cache_attention(c.cache, q[:0], out[:0], table, lengths)  # no rows: nothing to do
    starts = to_gpu(np.arange(5, dtype=np.int32))
    backend.cache_attention(c.cache, q, out, table, lengths, starts=starts, max_tokens=0)  # no row below the bound
    backend.sync()
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_a_bound_above_the_rows_there_are(backend, dtype):
    """A constant bound, as a caller keeps for its steps, on a step that brings less."""
    c = Case([300, 41, 17], [3, 1, 1], kv=2, group=3, dtype=dtype, page=16, seed=33)
    want = c.run(backend)
    c.check(want)
    for bound in (5, 8, 100, 2**32 - 1):
        assert np.array_equal(c.run(backend, max_tokens=bound), want)
    long = Case([700, 800], [100, 90], kv=1, group=4, dtype=dtype, page=16, seed=34)
    long.check(long.run(backend, max_tokens=4096, table=prompt_table(long)))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("tokens,length", [(1, 1), (3, 3), (3, 700), (70, 90)])
def test_queries_that_are_not_finite(backend, dtype, value, tokens, length):
    """NaN for the rows and heads that hold one, whatever the signs of the scores; zeros where such a row
    sees nothing; the others untouched."""
    c = Case([length, 0], [tokens, tokens], kv=2, group=2, d=64, page=16, dtype=dtype, seed=35)
    kw = dict(table=prompt_table(c)) if tokens * c.group > 64 else {}
    want = c.run(backend, **kw)
    c.check(want)
    hit = np.zeros((2 * tokens, 4), bool)
    for row, head, dim in ((0, 0, 0), (0, 3, 63), (tokens - 1, 1, 20), (tokens, 2, 7)):
        c.q[row, head, dim] = value
        hit[row, head] = row < tokens
    got = c.run(backend, **kw)
    assert np.array_equal(np.isnan(got).all(-1), hit) and np.array_equal(np.isnan(got).any(-1), hit)
    assert np.array_equal(got[~hit], want[~hit])
    assert not got[tokens:].any()
