"""Attention over the quantised cache on cuda:0 against the float64 oracle
(oracle/cache_oracle.py), which is given the values the cache stands for.

Bounds, derived from the arithmetic (include/nuq.h, nuq_cache_attention):
  * a score is off by at most delta = 2^-20 * max_j scale * sum|q k_j|: queries
    hold 22 bits (F16: all), products are exact and their F32 sums of at most
    256 terms, the scaling and the subtraction round to 24 bits each;
  * a weight is then off by a relative 2 delta (its own and the sum's), 2^-19 for
    the F32 sums over tokens and the exponential, and, F16 only, 2^-11 for its
    rounding to f16; below f16's normal range it is off by at most 2^-24 of
    the row's sum instead;
  * so |o - ref| <= (2 delta + 2^-19 [+ 2^-11]) * sum p|v| + 2^-24 * sum|v|,
    and F16 outputs round once more: 2^-11 |ref| + 2^-25.
"""
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


class Case:
    """Sequences of lengths `held` that bring `brought` tokens, in a shuffled cache whose
    unwritten places hold ones in every bit (NaN scales)."""

    def __init__(self, held, brought, bits=4, d=128, page=64, kv=2, group=6, dtype="f32", seed=0, spread=1.5):
        import torch
        self.rng = rng = np.random.default_rng(seed)
        self.held, self.brought = held, brought
        self.d, self.kv, self.group, self.page = d, kv, group, page
        need = [max(1, -(-n // page)) for n in held]
        pages = sum(need) + 2
        self.cache = nq.KVCache(bits, pages, page, kv, d)
        self.cache.bytes.fill_(255)
        order = rng.permutation(pages)
        self.table = np.full((len(held), max(need) + 1), pages + 7, np.int32)  # unused entries name no page
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k, self.v = [], []
        backend = nq.Backend(0)
        for b, n in enumerate(held):
            k = (rng.standard_normal((n, kv, d)) * np.exp(0.5 * rng.standard_normal((1, kv, d)))).astype(np.float32)
            v = (rng.standard_normal((n, kv, d)) + 0.3).astype(np.float32)
            self.k.append(k), self.v.append(v)
            if n:
                self.write(backend, b, k, v)
        backend.sync()
        backend.close()
        rows = sum(brought)
        self.q = (rng.standard_normal((rows, kv * group, d)) * spread).astype(np.float32)
        self.dtype = torch.float32 if dtype == "f32" else torch.float16
        if dtype == "f16":
            self.q = self.q.astype(np.float16)
        self.bits = bits

    def slots(self, b, positions):
        return (self.table[b, positions // self.page].astype(np.int64) * self.page + positions % self.page)

    def write(self, backend, b, k, v):
        import torch
        backend.cache_write(self.cache, to_gpu(k), to_gpu(v), to_gpu(self.slots(b, np.arange(len(k)))))
        torch.cuda.synchronize()
        want = co.stored(self.cache.bits, k, v)
        if not hasattr(self, "values"):
            self.values = {}
        self.values[b] = want[:2]

    def run(self, backend, window=0, scale=None, starts=None, table=None, lengths=None, out=None, q=None, **more):
        import torch
        q = to_gpu(self.q) if q is None else q
        out = torch.full(q.shape, 7.0, dtype=self.dtype, device="cuda") if out is None else out
        if starts is None and len(set(self.brought)) > 1:
            starts = np.concatenate([[0], np.cumsum(self.brought)])
        backend.cache_attention(self.cache, q, out, to_gpu(self.table if table is None else table),
                                to_gpu(np.array(self.held if lengths is None else lengths, np.int32)),
                                starts=None if starts is None else to_gpu(starts.astype(np.int32)), window=window,
                                scale=scale, **more)
        backend.sync()
        return out.float().cpu().numpy().astype(np.float64)

    def check(self, got, window=0, scale=None, absent=None, rows=None):
        scale = self.d ** -0.5 if scale is None else scale
        at, worst = 0, 0.0
        for b, (n, new) in enumerate(zip(self.held, self.brought)):
            pick = np.arange(new) if rows is None else np.unique(np.clip(rows, 0, new - 1))
            for i in pick:
                k, v = self.values.get(b, (np.zeros((0, self.kv, self.d)),) * 2)
                o, mass, plain, reach = co.attention(self.q[at + i:at + i + 1], k, v, n - new + i, self.group, scale,
                                                     window, None if absent is None else absent.get(b))
                f16 = self.dtype.itemsize == 2
                delta = 2.0 ** -20 * reach[..., None]
                bound = (2 * delta + 2.0 ** -19 + (2.0 ** -11 if f16 else 0)) * mass + 2.0 ** -24 * plain
                bound += (2.0 ** -11 * np.abs(o) + 2.0 ** -25) if f16 else 1e-37
                g = got[at + i:at + i + 1]
                assert np.array_equal(np.isnan(g), np.isnan(o)), (b, i)
                err = np.where(np.isnan(o), 0, np.abs(g - o))
                assert np.all(err <= np.where(np.isnan(o), 1, bound)), (b, i, np.nanmax(err / bound))
                worst = max(worst, float(np.nanmax(np.where(np.isnan(o), 0, err / np.where(np.isnan(o), 1, bound)))))
            at += new
        print(f"worst share of the bound {worst:.3f}")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,page,kv,group", [(128, 64, 2, 6), (64, 16, 1, 1), (256, 32, 3, 2), (128, 16, 1, 16)])
@pytest.mark.parametrize("length", [1, 15, 33, 700])
def test_one_token(backend, dtype, bits, d, page, kv, group, length):
    print(f"[attention] one token {dtype} bits {bits} d {d} page {page} kv {kv} group {group} length {length}", flush=True)
    c = Case([length], [1], bits, d, page, kv, group, dtype, seed=length + d)
    c.check(c.run(backend))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d,bits", [(128, 4), (64, 8), (256, 4), (256, 8)])
@pytest.mark.parametrize("tokens,length", [(2, 2), (3, 130), (8, 517), (11, 40), (65, 65), (130, 301)])
def test_several_tokens(backend, dtype, d, bits, tokens, length):
    print(f"[attention] {tokens} tokens {dtype} d {d} bits {bits} length {length}", flush=True)
    c = Case([length], [tokens], bits, d, 32, 2, 3, dtype, seed=tokens)
    c.check(c.run(backend))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 5, 32, 100, 10000])
@pytest.mark.parametrize("tokens", [1, 7, 90])
def test_sliding_window(backend, dtype, window, tokens):
    print(f"[attention] window {window} tokens {tokens} {dtype}", flush=True)
    c = Case([433, 95], [tokens, tokens], dtype=dtype, page=16, kv=1, group=4, seed=window)
    c.check(c.run(backend, window=window), window=window)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_ragged_batch_with_empty_sequences(backend, dtype):
    """Counts of 0 to 40 new tokens, a sequence of length 0, one shorter than what
    it is said to bring: rows that see nothing are zeros."""
    c = Case([300, 0, 17, 1, 64, 500], [5, 1, 40, 1, 0, 33], dtype=dtype, kv=2, group=3, d=64, page=16, seed=3)
    got = c.run(backend)
    c.check(got)
    assert not got[5].any()          # the empty sequence
    assert not got[6:6 + 23].any()   # positions before the third one's start


def test_long_axis_split_over_workgroups(backend):
    for dtype in ("f32", "f16"):
        c = Case([9001], [1], dtype=dtype, kv=1, group=5, seed=4)
        split = c.run(backend)
        c.check(split)
        whole = c.run(backend, max_length=1)  # a bound of one step: one workgroup a head
        c.check(whole)


def test_poisoned_tokens_reach_only_the_rows_that_see_them(backend):
    """A NaN in K of one token and in V of another; rows before them and rows whose
    window has passed them are untouched."""
    import torch
    for dtype in ("f32", "f16"):
        c = Case([200], [100], dtype=dtype, kv=2, group=2, d=64, page=16, seed=5)
        c.k[0][130, 0, 3] = np.nan
        c.v[0][140, 1, 60] = np.inf
        c.write(backend, 0, c.k[0], c.v[0])
        torch.cuda.synchronize()
        got = c.run(backend, window=20)
        c.check(got, window=20)
        nan = np.isnan(got).any(-1)
        assert nan[30:50, :2].all() and not nan[30:50, 2:][:10].any() and nan[40:60, 2:].all()
        assert not nan[:30].any() and not nan[60:].any()


def test_positions_on_missing_pages_are_not_attended_to(backend):
    for dtype in ("f32", "f16"):
        c = Case([150], [20], dtype=dtype, kv=2, group=2, page=16, seed=6)
        table = c.table.copy()
        table[0, 2], table[0, 5] = -1, 1 << 30
        absent = np.zeros(150, bool)
        absent[32:48] = absent[80:96] = True
        c.check(c.run(backend, table=table), absent={0: absent})
        table[0, :] = -1
        assert not c.run(backend, table=table).any()


def test_lengths_past_the_table_and_negative_ones(backend):
    c = Case([64], [4], kv=1, group=2, page=16, d=64, seed=7)
    full = c.run(backend, table=c.table[:, :4])
    assert np.array_equal(c.run(backend, table=c.table[:, :4], lengths=[1 << 30]), full)
    assert not c.run(backend, lengths=[-5]).any()


def test_rows_no_sequence_has_stay_as_they_are(backend):
    """starts that leave rows out, run backwards or past the end, and a bound on the rows of a sequence."""
    c = Case([40, 50], [4, 4], kv=1, group=2, d=64, page=16, seed=8)
    want = c.run(backend)
    got = c.run(backend, starts=np.array([0, 4, 4]), lengths=[40, 50])
    assert np.array_equal(got[:4], want[:4]) and np.all(got[4:] == 7.0)
    got = c.run(backend, starts=np.array([6, 2, 1000]), lengths=[40, 54])
    assert np.all(got[:2] == 7.0) and not np.any(got[2:] == 7.0)
    got = c.run(backend, starts=np.array([0, 4, 8]), max_tokens=2, lengths=[38, 48])
    assert np.all(got[2:4] == 7.0) and np.all(got[6:] == 7.0) and np.array_equal(got[:2], want[:2])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strided_queries_and_outputs(backend, dtype):
    """Queries inside a merged q/k/v row, outputs inside a wider buffer."""
    import torch
    c = Case([90, 77], [3, 3], dtype=dtype, kv=2, group=2, seed=9)
    want = c.run(backend)
    wide = torch.full((6, 8, 128), 3.0, dtype=c.dtype, device="cuda")
    wide[:, :4] = to_gpu(c.q)
    out = torch.full((6, 7, 128), 7.0, dtype=c.dtype, device="cuda")
    got = c.run(backend, q=wide[:, :4], out=out[:, :4])
    assert np.array_equal(got, want) and bool((out[:, 4:] == 7.0).all())


def test_queries_of_any_magnitude_keep_f32_precision(backend):
    """Rows scaled by powers of ten, the scale undoing it: the same weights."""
    c = Case([300], [1], kv=1, group=8, seed=10)
    for factor in (1e-30, 1e-6, 1e4, 1e30):
        c2 = Case([300], [1], kv=1, group=8, seed=10)
        c2.q = (c.q.astype(np.float64) * factor).astype(np.float32)
        c2.check(c2.run(backend, scale=128 ** -0.5 / factor), scale=float(np.float32(128 ** -0.5 / factor)))


def test_large_scores_do_not_overflow(backend):
    """Scores in the thousands: the softmax is a selection."""
    for dtype in ("f32", "f16"):
        c = Case([500], [9], dtype=dtype, kv=1, group=2, seed=11, spread=300.0)
        c.check(c.run(backend))


def test_the_same_call_gives_the_same_bits(backend):
    c = Case([5000, 1234], [2, 2], kv=2, group=6, seed=12)
    assert np.array_equal(c.run(backend), c.run(backend))


def test_graph_capture_without_and_with_a_workspace():
    """Captured on a fresh context (fewer splits, no allocation) and again after the
    eager call grew its workspace; replays equal the eager result to rounding, with other work between."""
    import torch
    c = Case([6000], [1], kv=1, group=4, seed=13)
    b = nq.Backend(0)
    q, table = to_gpu(c.q), to_gpu(c.table)
    lengths = to_gpu(np.array([6000], np.int32))
    stream = torch.cuda.Stream()
    eager = None
    for _ in range(2):
        out = torch.zeros(1, 4, 128, device="cuda")
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            b.cache_attention(c.cache, q, out, table, lengths)
        for _ in range(3):
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c.check(out.cpu().numpy().astype(np.float64))
            eager = c.run(b)
        c.check(eager)
    assert np.array_equal(out.cpu().numpy(), eager.astype(np.float32))
    b.close()


def test_refusals_leave_the_output_untouched(backend):
    import torch
    c = Case([40, 50], [2, 2], kv=2, group=2, d=64, page=16, seed=14)
    q, table, lengths = to_gpu(c.q), to_gpu(c.table), to_gpu(np.array([40, 50], np.int32))
    out = torch.full(q.shape, 7.0, device="cuda")
    cases = [
        (dict(q=q[:, :3]), nq.InvalidShape),                       # 3 query heads over 2
        (dict(q=q[:3]), nq.InvalidShape), (dict(output=out.half()), nq.InvalidShape),
        (dict(q=q.double(), output=out.double()), nq.InvalidArgument),
        (dict(q=q[..., :32], output=out[..., :32]), nq.InvalidShape),
        (dict(page_table=table.long()), nq.InvalidArgument), (dict(page_table=table[:1]), nq.InvalidShape),
        (dict(page_table=table[:, :0]), nq.InvalidShape),
        (dict(lengths=lengths.long()), nq.InvalidArgument),
        (dict(starts=to_gpu(np.array([0, 4], np.int32))), nq.InvalidShape),
        (dict(scale=0.0), nq.InvalidShape), (dict(scale=float("nan")), nq.InvalidShape),
        (dict(scale=-1.0), nq.InvalidShape), (dict(scale=float("inf")), nq.InvalidShape),
        (dict(max_tokens=3), nq.InvalidShape), (dict(max_tokens=5), nq.InvalidShape),
        (dict(window=-1), nq.InvalidShape), (dict(max_tokens=-1), nq.InvalidShape), (dict(max_length=-1), nq.InvalidShape),
    ]
    for change, error in cases:
        args = dict(cache=c.cache, q=q, output=out, page_table=table, lengths=lengths, **{})
        if "q" in change and "output" not in change:
            args["output"] = torch.empty_like(change["q"]) if change["q"].shape[0] == 4 else out
        args.update(change)
        with pytest.raises(error):
            backend.cache_attention(**args)
    backend.sync()
    assert bool((out == 7.0).all())
    empty = torch.empty(0, 4, 64, device="cuda")
    backend.cache_attention(c.cache, empty, empty, table[:0], lengths[:0])  # nothing to do


def prompt_table(c):
    """The case's page table with so many more entries, none of which names a page, that the
    tokens its rows could see make it a prompt's work: the kernel that decodes the
    cache once for four waves takes it, split over workgroups, however short it is."""
    brought, heads = max(c.brought), c.kv * c.group
    assert brought * c.group > 64
    wide = -(-int(1.3e10 / (sum(c.brought) * heads * c.d)) // c.page) + 1
    table = np.full((len(c.held), max(wide, c.table.shape[1])), -1, np.int32)
    table[:, :c.table.shape[1]] = c.table
    return table


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,page,kv,group", [(64, 16, 1, 3), (128, 64, 2, 6), (256, 32, 1, 5)])
@pytest.mark.parametrize("tokens,length", [(22, 22), (65, 65), (66, 130), (70, 531)])
def test_prompt_rows(backend, dtype, bits, d, page, kv, group, tokens, length):
    print(f"[attention] prompt {dtype} bits {bits} d {d} kv {kv} group {group} tokens {tokens} length {length}", flush=True)
    c = Case([length], [tokens], bits, d, page, kv, group, dtype, seed=tokens + d)
    c.check(c.run(backend, table=prompt_table(c)))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_rows_of_ragged_and_empty_sequences(backend, dtype, d):
    c = Case([300, 0, 17, 1, 64, 500], [35, 1, 40, 1, 0, 33], dtype=dtype, kv=2, group=3, d=d, page=16, seed=15)
    got = c.run(backend, table=prompt_table(c))
    c.check(got)
    assert not got[35].any()          # the empty sequence
    assert not got[36:36 + 23].any()  # positions before the third one's start


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_prompt_rows_and_poisoned_tokens(backend, dtype, bits):
    import torch
    c = Case([200], [100], bits, dtype=dtype, kv=2, group=2, d=64, page=16, seed=16)
    c.k[0][130, 0, 3] = np.nan
    c.v[0][140, 1, 60] = np.inf
    c.write(backend, 0, c.k[0], c.v[0])
    torch.cuda.synchronize()
    got = c.run(backend, table=prompt_table(c))
    c.check(got)
    nan = np.isnan(got).any(-1)
    assert not nan[:30, :2].any() and nan[30:, :2].all() and not nan[:40, 2:].any() and nan[40:, 2:].all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d,bits", [(64, 8), (128, 4), (256, 4)])
def test_prompt_rows_and_missing_pages(backend, dtype, d, bits):
    c = Case([150], [40], bits, dtype=dtype, kv=2, group=2, d=d, page=16, seed=17)
    table = prompt_table(c)
    table[0, 2], table[0, 5] = -1, 1 << 30
    absent = np.zeros(150, bool)
    absent[32:48] = absent[80:96] = True
    c.check(c.run(backend, table=table), absent={0: absent})
    table[0, 1:] = -1
    absent[16:] = True
    c.check(c.run(backend, table=table), absent={0: absent})  # whole steps and splits without a page
    table[0, 0] = -1
    assert not c.run(backend, table=table).any()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_prompt_rows_large_scores_strides_and_rows_no_sequence_has(backend, dtype):
    import torch
    c = Case([500, 90], [40, 40], dtype=dtype, kv=1, group=3, page=16, seed=18, spread=300.0)
    table = prompt_table(c)
    want = c.run(backend, table=table)
    c.check(want)
    wide = torch.full((80, 8, 128), 3.0, dtype=c.dtype, device="cuda")
    wide[:, :3] = to_gpu(c.q)
    out = torch.full((80, 7, 128), 7.0, dtype=c.dtype, device="cuda")
    got = c.run(backend, table=table, q=wide[:, :3], out=out[:, :3])
    assert np.array_equal(got, want) and bool((out[:, 3:] == 7.0).all())
    got = c.run(backend, table=table, starts=np.array([0, 40, 70]), lengths=[500, 80])
    assert np.array_equal(got[:70], want[:70]) and np.all(got[70:] == 7.0)
    got = c.run(backend, table=table, starts=np.array([10, 5, 1000]), lengths=[500, 125])
    assert np.all(got[:5] == 7.0) and not np.any(got[5:] == 7.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d,bits,kv,group", [(64, 4, 2, 50), (128, 4, 8, 6), (128, 8, 1, 48), (256, 4, 4, 24)])
@pytest.mark.parametrize("window", [0, 33])
def test_long_prompts(backend, dtype, d, bits, kv, group, window):
    """A prompt long enough by itself, one workgroup along the axis (D = 256 splits
    without a window), on rows at the edges of steps, tiles and the prompt."""
    print(f"[attention] long prompt {dtype} d {d} bits {bits} kv {kv} group {group} window {window}", flush=True)
    c = Case([2185], [2151], bits, d, 32, kv, group, dtype, seed=19)
    rows = [0, 1, 29, 30, 31, 32, 33, 34, 62, 63, 64, 65, 94, 95, 97, 128, 500, 1023, 1024, 1999, 2013, 2014, 2149, 2150]
    c.check(c.run(backend, window=window), window=window, rows=rows)
    assert np.isfinite(c.run(backend, window=window)).all()


def test_prompt_rows_replayed_from_a_graph(backend):
    import torch
    c = Case([700], [50], kv=2, group=2, seed=20)
    b = nq.Backend(0)
    q, table, lengths = to_gpu(c.q), to_gpu(prompt_table(c)), to_gpu(np.array([700], np.int32))
    stream, out = torch.cuda.Stream(), torch.zeros(50, 4, 128, device="cuda")
    for _ in range(2):  # without a workspace, then with one
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            b.cache_attention(c.cache, q, out, table, lengths)
        for _ in range(3):
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c.check(out.cpu().numpy().astype(np.float64))
            c.run(b, table=prompt_table(c))
    b.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d,kv,group,lengths,tokens", [(64, 2, 5, [1900, 0, 3100], [3, 1, 2]), (128, 1, 3, [2500, 2499], [1, 1]),
                                                       (256, 4, 2, [4100, 40], [5, 3]), (128, 8, 6, [3000] * 9, [2] * 9)])
def test_few_and_many_splits_of_ragged_rows(backend, dtype, d, kv, group, lengths, tokens):
    """Axes split by a few (bounds on the length that ask for 2 to 8) and by many, with splits that hold
    nothing of the short sequences."""
    c = Case(lengths, tokens, 4, d, 32, kv, group, dtype, seed=21)
    for bound in (0, 200, 600, 1000, 2100):
        c.check(c.run(backend, max_length=bound))


def test_a_prompt_among_many_single_tokens(backend):
    """One call for a long prompt and hundreds of sequences that bring a token each."""
    c = Case([1000] + [5] * 399, [1000] + [1] * 399, d=64, kv=1, group=48, page=16, dtype="f16", seed=22)
    c.check(c.run(backend), rows=[0, 1, 63, 64, 511, 998, 999])


@pytest.mark.parametrize("tokens", [2, 70])
def test_offsets_past_32_bits(backend, tokens):
    """Pages beyond 4 GiB of a cache, and query and output rows beyond 2^32 bytes of their buffers,
    give what the same tokens give near their starts, by rows and as a prompt."""
    import torch
    c = Case([131], [tokens], kv=8, group=1, page=64, dtype="f16", seed=23)
    table = c.table if tokens < 64 else prompt_table(c)
    want = c.run(backend, table=table)
    c.check(want)
    pages = (1 << 32) // (64 * 8 * 144) + 8
    far = nq.KVCache(4, pages, 64, 8, 128)
    page_bytes = 64 * 8 * 144
    moved = np.where((table >= 0) & (table < c.cache.pages), table + pages - c.cache.pages, -1).astype(np.int32)
    far.bytes[(pages - c.cache.pages) * page_bytes:] = c.cache.bytes
    c.cache = far
    assert np.array_equal(c.run(backend, table=moved), want)
    stride = (1 << 32) // (2 * (tokens - 1)) // 8 * 8 + 1024
    held = torch.empty(2, (tokens - 1) * stride + 1024, dtype=torch.float16, device="cuda")
    q, out = (h.as_strided((tokens, 8, 128), (stride, 128, 1)) for h in held)
    q.copy_(to_gpu(c.q))
    out.fill_(7.0)
    assert np.array_equal(c.run(backend, table=moved, q=q, out=out), want)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d,kv,group", [(64, 1, 6), (128, 2, 3), (256, 1, 12)])
def test_prompts_among_single_tokens_and_drafts(backend, dtype, d, kv, group):
    """More sequences than a wave has lanes, some of many tokens, some of one, a few or none, each
    kind with its own splits and partial results."""
    rng = np.random.default_rng(24)
    brought = [1] * 85
    brought[3], brought[40], brought[66], brought[84] = 130, 64 // group + 1, 77, 64 // group
    brought[10] = brought[64] = 0
    held = [int(n) for n in rng.integers(1, 400, 85)]
    held[3], held[5], held[66], held[70], held[84] = 700, 0, 77, 1500, 900
    c = Case(held, brought, d=d, kv=kv, group=group, page=16, dtype=dtype, seed=25)
    got = c.run(backend, table=prompt_table(c))
    c.check(got)
    c.check(c.run(backend, window=150), window=150)
