"""Sequences through a dense layer and lm_head over the quantised K/V cache: the
layer of layer.py (same projections, residuals and SiLU pair; norms and rotary
positions omitted there and here) past the first position, for prompts, chunks of
them and decoded tokens of several sequences in one step:

  q, k, v = W_q x, W_k x, W_v x       the new tokens' rows
  cache[slots] = k, v                 Backend.cache_write
  a = attention(q, cache)             Backend.cache_attention
  h1 = x + W_o a
  h2 = h1 + W_down * (silu(W_gate * h1) * (W_up * h1))
  logits = W_lm_head * h2
  score(): log p(token), entropy and alternatives   Backend.logprobs

All projections, the cache and the attention run in libnuq.so; torch holds the
buffers and adds. Pages are handed out as sequences grow and come back with
`release`; the host keeps the lengths, so a step asks the GPU nothing and waits for
nothing: steps queue behind each other (but where a buffer or the workspace grows).
"""
from __future__ import annotations

import numpy as np

from . import backend as nb


class CachedLayer:
    """mats: the layer's matrices by layer.SHAPES' names, of any sizes whose query
    and key rows are whole heads. Holds up to `sequences` sequences and `pages`
    pages of `page_tokens` tokens."""

    def __init__(self, backend: nb.Backend, mats: dict, sequences: int, pages: int, page_tokens: int = 64,
                 bits: int = 4, head_dim: int = 128, window: int = 0):
        import torch
        self._torch, self.backend, self.mats, self.window = torch, backend, mats, window
        self.q_rows, self.kv_rows, self.hidden = mats["q"].rows, mats["k"].rows, mats["q"].columns
        ffn = mats["gate"].rows
        fit = {"q": (self.q_rows, self.hidden), "k": (self.kv_rows, self.hidden), "v": (self.kv_rows, self.hidden),
               "o": (self.hidden, self.q_rows), "gate": (ffn, self.hidden), "up": (ffn, self.hidden),
               "down": (self.hidden, ffn), "lm_head": (mats["lm_head"].rows, self.hidden)}
        for name, (rows, columns) in fit.items():
            if (mats[name].rows, mats[name].columns) != (rows, columns):
                raise nb.InvalidShape(f"InvalidShape: {name} is {mats[name].rows} x {mats[name].columns}, "
                                      f"not {rows} x {columns}")
        if self.kv_rows % head_dim or self.q_rows % self.kv_rows:
            raise nb.InvalidShape(f"InvalidShape: {self.q_rows} and {self.kv_rows} rows are not whole heads of {head_dim}")
        self.head_dim = head_dim
        self.cache = nb.KVCache(bits, pages, page_tokens, self.kv_rows // head_dim, head_dim, device=backend.device)
        self.lengths = [0] * sequences
        self.free = list(range(pages))[::-1]
        self.pages = [[] for _ in range(sequences)]
        self.table = np.full((sequences, pages), -1, np.int32)  # host copy of what the GPU is given
        self.buffers = {}

    def _buffer(self, name: str, rows: int, columns: int):
        held = self.buffers.get(name)
        if held is None or held.shape[0] < rows:
            held = self.buffers[name] = self._torch.empty(rows, columns, device=f"cuda:{self.backend.device}")
        return held[:rows]

    def release(self, sequence: int) -> None:
        """Ends a sequence: its pages are free for others."""
        self.free += self.pages[sequence][::-1]
        self.pages[sequence], self.lengths[sequence] = [], 0
        self.table[sequence] = -1

    def _grow(self, counts) -> np.ndarray:
        """Gives the sequences room for their new tokens and returns these tokens' slots."""
        page = self.cache.page_tokens
        wanted = [-(-(n + c) // page) - len(p) for n, c, p in zip(self.lengths, counts, self.pages)]
        if sum(wanted) > len(self.free):
            raise nb.InvalidShape(f"InvalidShape: {sum(wanted)} pages wanted, {len(self.free)} free")
        slots = []
        for b, (more, count) in enumerate(zip(wanted, counts)):
            for _ in range(more):
                self.table[b, len(self.pages[b])] = self.free[-1]
                self.pages[b].append(self.free.pop())
            at = np.arange(self.lengths[b], self.lengths[b] + count)
            slots.append(self.table[b, at // page].astype(np.int64) * page + at % page)
            self.lengths[b] += count
        return np.concatenate(slots)

    def _shrink(self, lengths) -> None:
        """Takes a step back: the sequences hold `lengths` tokens again, and the pages past them are free, in
        the order they were in."""
        for b in reversed(range(len(lengths))):
            keep = -(-lengths[b] // self.cache.page_tokens)
            while len(self.pages[b]) > keep:
                self.free.append(self.pages[b].pop())
                self.table[b, len(self.pages[b])] = -1
            self.lengths[b] = lengths[b]

    def _device(self, array):
        """The array on the GPU, by a copy that is queued: from pageable memory it would wait for all work
        before it. (Pinned blocks come from torch's pool, which keeps them until their copy is done.)"""
        torch = self._torch
        if torch.cuda.is_current_stream_capturing():
            raise nb.InvalidArgument("a step's tables and lengths come from the host: a graph would replay this step's")
        array = torch.from_numpy(np.ascontiguousarray(array))
        held = torch.empty(array.shape, dtype=array.dtype, pin_memory=True)
        return held.copy_(array).to(f"cuda:{self.backend.device}", non_blocking=True)

    def _project(self, name: str, x, out) -> None:
        self.backend.matmul(self.mats[name], x, x.stride(0), out, out.stride(0), x.shape[0])

    def forward(self, x, counts):
        """x [sum(counts)][hidden] F32, rows contiguous: every sequence's new tokens (counts[b], 0 for a
        sequence that rests), one sequence's behind the other's. Returns the
        logits [sum(counts)][vocabulary], good until the next call. If it raises, the sequences hold
        what they held before."""
        rows = int(sum(counts))
        if len(counts) != len(self.lengths) or min(counts, default=0) < 0 or tuple(x.shape) != (rows, self.hidden):
            raise nb.InvalidShape(f"InvalidShape: {len(counts)} counts of {len(self.lengths)} sequences, "
                                  f"{rows} rows, x {tuple(x.shape)}")
        if x.dtype is not self._torch.float32 or x.get_device() != self.backend.device:
            raise nb.InvalidArgument(f"x is {x.dtype} on {x.device}, not float32 on cuda:{self.backend.device}")
        if self.hidden > 1 and x.stride(1) != 1:
            raise nb.InvalidShape(f"InvalidShape: x's rows are not contiguous (strides {x.stride()})")
        if rows == 0:
            return self._buffer("logits", 0, self.mats["lm_head"].rows)
        before = list(self.lengths)
        try:
            return self._step(x, counts, rows, self._device(self._grow(counts)))
        except BaseException:
            self._shrink(before)  # a step that failed has not happened: it can be tried again
            raise

    def _step(self, x, counts, rows: int, slots):
        torch, b, m = self._torch, self.backend, self.mats
        q_rows, kv_rows, single = self.q_rows, self.kv_rows, rows == 1
        qkv = self._buffer("qkv", rows, q_rows + 2 * kv_rows)
        q, k, v = qkv[:, :q_rows], qkv[:, q_rows:q_rows + kv_rows], qkv[:, q_rows + kv_rows:]
        if single:
            b.matvec_segments([(m["q"], q), (m["k"], k), (m["v"], v)], x, nb.SEGMENT_PLAIN)
        else:
            for name, out in (("q", q), ("k", k), ("v", v)):
                self._project(name, x, out)
        heads = lambda t: t.unflatten(1, (-1, self.head_dim))  # noqa: E731
        b.cache_write(self.cache, heads(k), heads(v), slots)
        attn = self._buffer("attn", rows, q_rows)
        most = max(len(p) for p in self.pages)
        equal = len(set(counts)) == 1
        b.cache_attention(self.cache, heads(q), heads(attn), self._device(self.table[:, :most]),
                          self._device(np.array(self.lengths, np.int32)),
                          starts=None if equal else self._device(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)),
                          window=self.window, max_tokens=max(counts), max_length=max(self.lengths))
        h1 = self._buffer("h1", rows, self.hidden)
        self._project("o", attn, h1)
        torch.add(h1, x, out=h1)
        act = self._buffer("act", rows, m["gate"].rows)
        if single:
            b.matvec_segments([(m["gate"], act), (m["up"], act)], h1, nb.SEGMENT_SILU_MUL_PAIR)
        else:
            up = self._buffer("up", rows, m["up"].rows)
            self._project("gate", h1, act)
            self._project("up", h1, up)
            torch.mul(torch.nn.functional.silu(act), up, out=act)
        h2 = self._buffer("h2", rows, self.hidden)
        self._project("down", act, h2)
        torch.add(h2, h1, out=h2)
        logits = self._buffer("logits", rows, m["lm_head"].rows)
        self._project("lm_head", h2, logits)
        return logits

    def score(self, logits, targets, top: int = 0):
        """Log probabilities of int32 targets [rows] under `logits`, the rows' entropies and, with
        `top`, the most probable tokens and their log probabilities: a dict of device tensors."""
        torch, rows, device = self._torch, logits.shape[0], logits.device
        out = {"logprobs": torch.empty(rows, device=device), "entropy": torch.empty(rows, device=device)}
        if top:
            out["top_ids"] = torch.empty(rows, top, dtype=torch.int32, device=device)
            out["top_logprobs"] = torch.empty(rows, top, device=device)
        self.backend.logprobs(logits, targets, *out.values())
        return out
