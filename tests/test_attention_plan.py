"""The attention's planner on the host (nuclis_amd/csrc/attention.hip): batches that a launch can take
have a plan, within the launch's limits. No GPU is used."""
import ctypes
import random

import pytest

import nuclis_amd as nq

MOST = 0xffffff  # workgroups of a launch
FIELDS = ("prompt", "splits", "groups", "join", "floats", "upto")


def plans(head_dim, kv_heads, heads, f32, rows, batch, max_tokens, ragged, max_length, window=0, max_floats=1 << 62, cus=256):
    f = nq.lib().nuq_attention_plan
    u32, u64 = ctypes.c_uint32, ctypes.c_uint64
    f.argtypes = [u32, u32, u32, u32, u32, u32, u32, ctypes.c_int, u64, u32, u64, u32, u64 * 12]
    out = (u64 * 12)()
    count = f(head_dim, kv_heads, heads, f32, rows, batch, max_tokens, ragged, max_length, window, max_floats, cus, out)
    return [dict(zip(FIELDS, out[6 * i:6 * i + 6])) for i in range(count)]


def check(found, where):
    for p in found:
        assert 1 <= p["splits"] <= 64 and 0 < p["groups"] <= MOST and p["join"] <= MOST, (where, p)
        assert (p["splits"] > 1) == (p["join"] > 0) == (p["floats"] > 0), (where, p)


@pytest.mark.parametrize("heads,batch,rows,max_tokens,length,f32", [
    (32, 256, 2303, 2048, 16384, 0),    # a chunk among single tokens
    (64, 128, 2175, 2048, 8192, 0),
    (48, 400, 1399, 1000, 16384, 0),
    (32, 128, 4223, 4096, 16384, 0),
    (64, 512, 512, 512, 8192, 0),       # single tokens under the loosest bound
    (48, 600, 600, 600, 4096, 1),
    (64, 4000, 4000, 4000, 128, 0),     # the same in short contexts
    (64, 4000, 4000, 4000, 128, 1),
])
def test_many_sequences_of_different_counts(heads, batch, rows, max_tokens, length, f32):
    check(plans(128, 8, heads, f32, rows, batch, max_tokens, 1, length), (heads, batch, rows, max_tokens, length, f32))


def test_plans_stay_within_a_launch():
    rng = random.Random(7)

    def log(low, high):
        return int(low * (high / low) ** rng.random())

    for _ in range(20000):
        kv = rng.choice([1, 2, 4, 8, 16])
        heads, d, f32 = kv * rng.choice([1, 2, 4, 6, 8, 16]), rng.choice([64, 128, 256]), rng.randint(0, 1)
        batch, most = log(1, 4000), log(1, 8000)
        length, window = log(most, 1 << 20), rng.choice([0, 0, log(1, 1 << 17)])
        floats = rng.choice([0, 1 << 20, 1 << 25, 1 << 62])
        if rng.random() < 0.7:
            rows = most + sum(rng.choice([1, 1, rng.randint(0, most)]) for _ in range(min(batch - 1, 50)))
            rows += max(0, batch - 51)
            if rng.random() < 0.3:
                most = rows  # no better bound than all rows
            ragged = 1
        else:
            rows, ragged = batch * most, 0
        if rows * heads > 1 << 27:
            continue
        where = (d, kv, heads, f32, rows, batch, most, ragged, length, window, floats)
        found = plans(*where)
        check(found, where)
        assert sum(p["floats"] for p in found) <= floats, (where, found)


def test_partial_results_of_a_call_stay_within_256_mib():
    """Both plans' together: a long chunk with wide heads among single tokens whose axes are split too."""
    found = plans(256, 1, 16, 0, 2055, 8, 2048, 1, 1 << 18)
    assert len(found) == 2 and all(p["splits"] > 1 for p in found)
    rng = random.Random(8)
    both = 0
    for _ in range(20000):
        kv, group, d = rng.choice([1, 1, 2, 4]), rng.choice([4, 8, 16]), rng.choice([64, 128, 256])
        batch, most = rng.randint(2, 12), rng.randint(300, 4000)
        found = plans(d, kv, kv * group, rng.randint(0, 1), most + batch - 1, batch, most, 1,
                      rng.choice([1 << 14, 1 << 16, 1 << 18]))
        both += len(found) == 2 and all(p["splits"] > 1 for p in found)
        assert 4 * sum(p["floats"] for p in found) <= 256 << 20, (kv, group, d, batch, most, found)
    assert both > 1000


@pytest.mark.parametrize("heads,rows,batch,tokens,length,f32,many,few", [
    (48, 1, 1, 1, 4096, 1, 32, 8),         # one token: a workgroup a compute unit
    (48, 32, 32, 1, 16384, 0, 4, 1),       # single tokens: four
    (48, 300, 1, 300, 16000, 0, 6, 3),     # a chunk, 80 workgroups: rounds of two
])
def test_splits_follow_the_compute_units(heads, rows, batch, tokens, length, f32, many, few):
    """The shape's splits on a whole device and on a quarter of one."""
    one = [plans(128, 8, heads, f32, rows, batch, tokens, 0, length, cus=cus)[0]["splits"] for cus in (256, 64)]
    assert one == [many, few]


def test_splits_of_wide_heads_follow_the_compute_units():
    splits = [plans(256, 4, 16, 0, 4096, 1, 4096, 0, 4096, cus=cus)[0]["splits"] for cus in (256, 64, 1024)]
    assert splits == [2, 1, 3]  # 512 workgroups; four splits' partial results would not fit
