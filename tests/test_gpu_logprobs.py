"""Log probabilities on cuda:0 against float64 (nuq_logprobs, include/nuq.h).

Bounds: x - m is exact to 2^-24 of |x - m|, e^(x-m) to a few 2^-24 more, and the F32
sums of at most 2^18 terms run over 16 in a thread, then a thread's steps (at most
64 here), then 64 lanes, waves and splits in a tree: ln z is off by at most
2^-16. So |lp - ref| <= 2^-16 + 2^-23 |ref|, and the entropy, whose terms have one
sign and whose sum carries the same relative error, by 2^-16 + 2^-15 ref. Ids are exact."""
import numpy as np
import pytest

import nuclis_amd as nq
from tests.gpu_util import to_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return nq.Backend(0)


def oracle(x, targets, top):
    x = x.astype(np.float64)
    rows, count = x.shape
    lp, entropy = np.full(rows, np.nan), np.zeros(rows)
    ids, tops = np.full((rows, top), -1, np.int64), np.full((rows, top), -np.inf)
    for r in range(rows):
        good = ~np.isnan(x[r])
        order = np.flatnonzero(good)[np.argsort(-x[r][good], kind="stable")][:top]
        ids[r, :len(order)] = order
        m = x[r].max()  # NaN where there is one
        if np.isneginf(m):
            ref, entropy[r] = np.full(count, -np.inf), 0.0
        else:
            with np.errstate(invalid="ignore"):
                d = x[r] - m
                z = np.exp(d).sum()
                ref = d - np.log(z)
                p = np.exp(ref)
                entropy[r] = -np.sum(np.where(p > 0, p * np.where(p > 0, ref, 0), p))
        if 0 <= targets[r] < count:
            lp[r] = ref[targets[r]]
        tops[r, :len(order)] = ref[order]
    return lp, entropy, ids, tops


def run(backend, x, targets, top, dtype="f32", pad=0):
    import torch
    t = to_gpu(x).to(torch.float16 if dtype == "f16" else torch.float32)
    rows, count = x.shape
    if pad:
        wide = torch.full((rows, count + pad), 99.0, dtype=t.dtype, device="cuda")  # larger than any logit
        wide[:, pad // 2:pad // 2 + count] = t
        t = wide[:, pad // 2:pad // 2 + count]
    lp, entropy = torch.full((rows,), 5.0, device="cuda"), torch.full((rows,), 5.0, device="cuda")
    ids = torch.full((rows, top), 5, dtype=torch.int32, device="cuda")
    tops = torch.full((rows, top), 5.0, device="cuda")
    backend.logprobs(t, to_gpu(np.asarray(targets, np.int32)), lp, entropy, ids, tops)
    backend.sync()
    return [v.cpu().numpy() for v in (lp, entropy, ids, tops)]


def check(got, want):
    for g, w, scale in ((got[0], want[0], 2.0 ** -23), (got[3], want[3], 2.0 ** -23), (got[1], want[1], 2.0 ** -15)):
        finite = np.isfinite(w)
        assert np.array_equal(g[~finite].astype(np.float64), w[~finite], equal_nan=True)
        assert np.all(np.abs(g[finite] - w[finite]) <= 2.0 ** -16 + scale * np.abs(w[finite]))
    assert np.array_equal(got[2], want[2])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,count,top", [(1, 1, 1), (1, 5, 5), (3, 64, 32), (2, 1000, 20), (7, 4097, 5), (1, 151936, 20),
                                            (5, 32003, 32), (300, 8191, 3), (1100, 513, 1), (2, 262144, 0)])
def test_rows_against_float64(backend, dtype, rows, count, top):
    print(f"[logprobs] {rows} x {count} top {top} {dtype}", flush=True)
    rng = np.random.default_rng(rows + count)
    x = (rng.standard_normal((rows, count)) * 3).astype(np.float32)
    x[:, rng.integers(0, count, 3)] += 6
    if dtype == "f16":
        x = x.astype(np.float16).astype(np.float32)  # ties throughout
    targets = rng.integers(0, count, rows)
    want = oracle(x, targets, top)
    check(run(backend, x, targets, top, dtype), want)
    if count > 1:
        check(run(backend, x, targets, top, dtype, pad=7), want)  # odd strides, rows off 16 bytes


def test_masked_ties_and_flat_rows(backend):
    rng = np.random.default_rng(3)
    count = 20011
    rows = np.stack([
        np.zeros(count), np.full(count, -np.inf), np.full(count, -3e38), np.arange(count) * 0.01,
        -np.arange(count) * 0.01, np.where(np.arange(count) % 2, 1.5, -np.inf),
        np.where(np.arange(count) == 77, 4.0, -np.inf), rng.integers(-3, 4, count).astype(float),
        np.where(np.arange(count) % 3, 0.0, -0.0), np.full(count, 3e38) * np.where(np.arange(count) % 5, 1, -1),
        np.where(np.arange(count) == 19999, 2e4, rng.standard_normal(count)),
        rng.standard_normal(count) * 1e-3 - 1e4]).astype(np.float32)
    targets = [5, 5, 5, 0, count - 1, 0, 77, 9, 3, 1, 19999, 4]
    for top in (1, 20, 32):
        check(run(backend, rows, targets, top), oracle(rows, targets, top))
    one = rows[[6]]
    check(run(backend, one, [1], 8), oracle(one, [1], 8))  # a single row, split over workgroups


def test_non_finite_rows_and_targets_outside(backend):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 9000)).astype(np.float32)
    x[0, 17] = np.nan
    x[1, 8999] = np.inf
    x[2, :] = np.nan
    x[3, 3:] = np.nan
    targets = [1, 1, 1, 0, -1, 9000]
    got, want = run(backend, x, targets, 5), oracle(x, targets, 5)
    assert np.isnan(got[0]).all()
    assert np.isnan(got[1][:4]).all() and np.array_equal(got[2], want[2])
    assert np.isnan(got[3][0]).all() and np.isnan(got[3][1]).all()
    assert np.all(got[2][2] == -1) and np.all(got[3][2] == -np.inf)
    assert got[2][3].tolist()[3:] == [-1, -1]
    check([g[4:] for g in got], [w[4:] for w in want])


def test_results_are_repeatable_and_need_no_alternatives(backend):
    import torch
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((4, 50000)) * 3).astype(np.float32)
    a, b = run(backend, x, [1, 2, 3, 4], 9), run(backend, x, [1, 2, 3, 4], 9)
    assert all(np.array_equal(p, q) for p, q in zip(a, b))
    lp, entropy = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    backend.logprobs(to_gpu(x), to_gpu(np.array([1, 2, 3, 4], np.int32)), lp, entropy)
    backend.sync()
    assert np.array_equal(lp.cpu().numpy(), a[0]) and np.array_equal(entropy.cpu().numpy(), a[1])


def test_graph_replays_on_a_fresh_context():
    """Captured before any workspace exists (a row is then one workgroup's), and after."""
    import torch
    b = nq.Backend(0)
    rng = np.random.default_rng(6)
    x = torch.zeros(2, 60000, device="cuda")
    targets = to_gpu(np.array([7, 59999], np.int32))
    out = [torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda"),
           torch.zeros(2, 6, dtype=torch.int32, device="cuda"), torch.zeros(2, 6, device="cuda")]
    stream = torch.cuda.Stream()
    for _ in range(2):
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            b.logprobs(x, targets, *out)
        for _ in range(3):
            v = (rng.standard_normal((2, 60000)) * 2).astype(np.float32)
            x.copy_(to_gpu(v))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            check([o.cpu().numpy() for o in out], oracle(v, [7, 59999], 6))
        run(b, v, [0, 1], 6)  # eager: the workspace grows
    b.close()


def test_refusals_leave_the_results_untouched(backend):
    import torch
    x = torch.zeros(3, 100, device="cuda")
    targets = torch.zeros(3, dtype=torch.int32, device="cuda")
    lp, entropy = torch.full((3,), 5.0, device="cuda"), torch.full((3,), 5.0, device="cuda")
    ids, tops = torch.full((3, 4), 5, dtype=torch.int32, device="cuda"), torch.full((3, 4), 5.0, device="cuda")
    wide = torch.full((3, 33), 5, dtype=torch.int32, device="cuda")
    for args, error in (((x[0], targets, lp, entropy), nq.InvalidShape), ((x.double(), targets, lp, entropy), nq.InvalidArgument),
                        ((x, targets.long(), lp, entropy), nq.InvalidArgument), ((x, targets[:2], lp, entropy), nq.InvalidShape),
                        ((x, targets, lp[:2], entropy), nq.InvalidShape), ((x.t(), targets, lp, entropy), nq.InvalidShape),
                        ((x, targets, lp, entropy, ids), nq.InvalidArgument),
                        ((x, targets, lp, entropy, ids, tops[:, :3]), nq.InvalidShape),
                        ((x, targets, lp, entropy, ids[:2], tops[:2]), nq.InvalidShape),
                        ((x, targets, lp, entropy, wide, wide.float()), nq.InvalidShape),
                        ((x[:, :3], targets, lp, entropy, ids, tops), nq.InvalidShape),
                        ((x[:, :0], targets, lp, entropy), nq.InvalidShape),
                        ((x[:1].expand(3, 100), targets, lp, entropy), nq.InvalidShape)):
        with pytest.raises(error):
            backend.logprobs(*args)
    backend.sync()
    assert bool((lp == 5).all()) and bool((entropy == 5).all()) and bool((ids == 5).all()) and bool((tops == 5).all())
    backend.logprobs(x[:0], targets[:0], lp[:0], entropy[:0])  # no rows: nothing to do


def test_rows_past_32_bits_of_bytes(backend):
    import torch
    x = (3 * np.random.default_rng(60).standard_normal((3, 5001))).astype(np.float32)
    stride = (1 << 30) + 3
    held = torch.empty(2 * stride + 5001, device="cuda")
    far = held.as_strided((3, 5001), (stride, 1))
    far.copy_(to_gpu(x))
    results = []
    for logits in (to_gpu(x), far):
        out = [torch.empty(3, device="cuda"), torch.empty(3, device="cuda"),
               torch.empty(3, 7, dtype=torch.int32, device="cuda"), torch.empty(3, 7, device="cuda")]
        backend.logprobs(logits, torch.tensor([1, 5000, 77], dtype=torch.int32, device="cuda"), *out)
        backend.sync()
        results.append([t.cpu().numpy() for t in out])
    near, far_ones = results
    order = np.argsort(-x, axis=1, kind="stable")[:, :7]
    assert np.array_equal(near[2], order) and np.array_equal(far_ones[2], order)
    for a, b in zip(near, far_ones):  # other alignments sum in another order: each within the bound above
        assert np.allclose(a, b, rtol=0, atol=2.0 ** -15)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_rows_in_order(backend, dtype, top):
    """Ascending rows, where every step beats all before it, and descending ones; a plateau at the bound."""
    x = np.sort(4 * np.random.default_rng(61).standard_normal((4, 70001)), axis=1).astype(np.float32)
    x[1] = x[1, ::-1]
    x[2] = np.minimum(x[2], 2.0)
    x[3] = np.round(x[3])
    if dtype == "f16":
        x = x.astype(np.float16).astype(np.float32)
    targets = np.array([0, 70000, 123, 69999])
    check(run(backend, x, targets, top, dtype), oracle(x, targets, top))
