"""Tensors that are not on the context's GPU never reach a call of the cache, attention and scoring
operators (nuclis_amd/backend.py). No GPU is used: the handle stands alone, and a tensor without
memory stands for one on the GPU."""
import pytest
import torch

import nuclis_amd as nq


class OnGpu:
    """A tensor of this shape and dtype that says it is on cuda:0."""

    def __init__(self, *shape, dtype=torch.float32, device=0):
        self._t, self._device = torch.empty(*shape, dtype=dtype, device="meta"), device

    def get_device(self):
        return self._device

    @property
    def device(self):
        return torch.device("cuda", self._device)

    def data_ptr(self):
        return 4096

    def __getattr__(self, name):
        return getattr(self._t, name)


@pytest.fixture
def handle(monkeypatch):
    b = object.__new__(nq.Backend)
    b._torch, b.device, b._h = torch, 0, None
    b._float_codes = {torch.float32: nq.F32, torch.float16: nq.F16}
    nq.lib()
    calls = []
    monkeypatch.setattr(b, "_call", lambda fn, *args: calls.append(fn))
    return b, calls


def host_of(t, device):
    return t._t.new_empty(t._t.shape, device="cpu") if device == "cpu" else OnGpu(*t.shape, dtype=t.dtype, device=1)


def refused_one_by_one(calls, call, args, device):
    call(**args)
    assert len(calls) == 1
    for name, value in args.items():
        elsewhere = dict(args)
        if isinstance(value, nq.KVCache):
            elsewhere[name] = nq.KVCache(4, 4, 16, 2, 64, bytes=host_of(value.bytes, device))
        elif isinstance(value, OnGpu):
            elsewhere[name] = host_of(value, device)
        else:
            continue
        with pytest.raises(nq.InvalidArgument, match="not cuda:0"):
            call(**elsewhere)
    assert len(calls) == 1


@pytest.mark.parametrize("device", ["cpu", "another GPU"])
def test_cache_calls(handle, device):
    b, calls = handle
    cache = nq.KVCache(4, 4, 16, 2, 64, bytes=OnGpu(nq.cache_bytes(4, 4, 16, 2, 64), dtype=torch.uint8))
    args = dict(cache=cache, k=OnGpu(3, 2, 64), v=OnGpu(3, 2, 64), slots=OnGpu(3, dtype=torch.int64))
    refused_one_by_one(calls, b.cache_write, args, device)
    calls.clear()
    refused_one_by_one(calls, b.cache_read, args, device)
    calls.clear()
    refused_one_by_one(calls, b.cache_attention, dict(
        cache=cache, q=OnGpu(3, 4, 64), output=OnGpu(3, 4, 64), page_table=OnGpu(2, 4, dtype=torch.int32),
        lengths=OnGpu(2, dtype=torch.int32), starts=OnGpu(3, dtype=torch.int32)), device)


@pytest.mark.parametrize("device", ["cpu", "another GPU"])
def test_logprobs(handle, device):
    b, calls = handle
    refused_one_by_one(calls, b.logprobs, dict(
        logits=OnGpu(3, 100), targets=OnGpu(3, dtype=torch.int32), logprobs=OnGpu(3), entropy=OnGpu(3),
        top_ids=OnGpu(3, 4, dtype=torch.int32), top_logprobs=OnGpu(3, 4)), device)
