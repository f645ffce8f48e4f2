"""Host-side mirror of nuclis's matmul backend over libnuq.so.

`Backend` keeps the method names, argument meaning and error behaviour of the
reference's Zig `Backend` for this path (inference/src/backends/metal/):
  matvec        ops/matvec.zig:32
  matvec_rows   ops/matvec.zig:149   (matvecRows)
  matvec_segments ops/matvec.zig:245 (matvecSegments)
  matmul        ops/matmul.zig:62
  matmul_kernel ops/matmul.zig:73    (matmulKernel)
  embed         ops/rowwise.zig:17
Errors are raised as the reference's typed errors (InvalidShape,
UnsupportedTensorEncoding, InvalidRowLength, InvalidByteLength,
NonFiniteResult). Every product runs in libnuq.so's HIP kernels; nothing here
computes. Device memory and streams come from PyTorch (plumbing only).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from pathlib import Path

import numpy as np

LIB_PATH = Path(__file__).resolve().parent / "libnuq.so"

Q8_0, Q4_K, Q5_K, Q6_K, IQ4_XS = 8, 12, 13, 14, 23
F32, F16 = 0, 1
KERNEL_AUTO, KERNEL_ROWS, KERNEL_TILE, KERNEL_GENERIC = 0, 1, 2, 3
SEGMENT_PLAIN, SEGMENT_SILU_MUL_PAIR = 0, 1
NOALLOC_MAX_PAIR_ROWS = 1 << 20  # NUQ_NOALLOC_MAX_PAIR_ROWS (include/nuq.h)

# inference/src/tensor/encoding.zig:29-41: id -> (values per block, bytes per block)
LAYOUT = {Q8_0: (32, 34), Q4_K: (256, 144), Q5_K: (256, 176), Q6_K: (256, 210), IQ4_XS: (256, 136)}


class NuqError(Exception):
    """Base of the typed errors; `.code` is the C status."""

    code = -1


class InvalidShape(NuqError):
    code = 1


class UnsupportedTensorEncoding(NuqError):
    code = 2


class InvalidRowLength(NuqError):
    code = 3


class InvalidByteLength(NuqError):
    code = 4


class NonFiniteResult(NuqError):
    code = 5


class DeviceError(NuqError):
    code = 6


class InvalidArgument(NuqError):
    code = 7


_ERRORS = {c.code: c for c in (InvalidShape, UnsupportedTensorEncoding, InvalidRowLength, InvalidByteLength,
                               NonFiniteResult, DeviceError, InvalidArgument)}


class _Matrix(ctypes.Structure):
    _fields_ = [("encoding", ctypes.c_uint32), ("reserved", ctypes.c_uint32), ("rows", ctypes.c_uint64),
                ("columns", ctypes.c_uint64), ("bytes", ctypes.c_void_p), ("byte_len", ctypes.c_uint64)]


class _TopKBuffers(ctypes.Structure):
    _fields_ = [("values", ctypes.c_void_p), ("indices", ctypes.c_void_p), ("sums", ctypes.c_void_p),
                ("flags", ctypes.c_void_p)]


# Backend.topk limits (backends/metal/ops/sampling.zig:15-22)
TOPK_CAPACITY, TOPK_PARTIALS, TOPK_MAX_COUNT = 256, 64, 262144


@dataclass
class TopK:
    """sampling.TopK (sampling/root.zig:154-173): the `count` best logits by
    (value descending, id ascending), Σ exp((l − max) / temperature) over every
    logit as the F64 sum of the device's F32 partial sums, and whether every
    logit was finite."""

    temperature: float
    ids: list
    values: list
    total: float
    finite: bool


class _Cache(ctypes.Structure):
    _fields_ = [("bits", ctypes.c_uint32), ("page_tokens", ctypes.c_uint32), ("kv_heads", ctypes.c_uint32),
                ("head_dim", ctypes.c_uint32), ("pages", ctypes.c_uint64), ("bytes", ctypes.c_void_p),
                ("byte_len", ctypes.c_uint64)]


class _Attention(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("dtype", ctypes.c_uint32),
                ("q_heads", ctypes.c_uint32), ("q_stride", ctypes.c_uint64), ("out_stride", ctypes.c_uint64),
                ("rows", ctypes.c_uint64), ("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_uint64),
                ("table_width", ctypes.c_uint64), ("lengths", ctypes.c_void_p), ("starts", ctypes.c_void_p),
                ("batch", ctypes.c_uint32), ("max_tokens", ctypes.c_uint32), ("max_length", ctypes.c_uint64),
                ("scale", ctypes.c_float), ("window", ctypes.c_uint32)]


class _Segment(ctypes.Structure):
    _fields_ = [("matrix", _Matrix), ("output", ctypes.c_void_p)]


_lib = None

EXPORTS = [
    "nuq_create", "nuq_destroy", "nuq_set_stream", "nuq_sync", "nuq_last_error", "nuq_set_generic_only",
    "nuq_validate_row", "nuq_embed", "nuq_dequant_range", "nuq_matvec", "nuq_matvec_rows", "nuq_matmul",
    "nuq_matmul_kernel", "nuq_matvec_segments", "nuq_argmax", "nuq_quantize_rows", "nuq_dequant_rows", "nuq_gemv",
    "nuq_gemm", "nuq_topk", "nuq_penalize", "nuq_reserve_workspace", "nuq_workspace_bytes",
    "nuq_matvec_segments_noalloc", "nuq_cache_bytes", "nuq_cache_write", "nuq_cache_read", "nuq_cache_attention",
    "nuq_logprobs",
]


def lib() -> ctypes.CDLL:
    """Loads libnuq.so; raises if it has not been built (no fallback exists)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
        # torch first: the library then binds to the HIP runtime that torch ships. The other way round the
        # process holds two of them, and whichever comes second finds no device.
        import torch  # noqa: F401
        L = ctypes.CDLL(str(LIB_PATH))
        vp, u32, u64 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64
        mp = ctypes.POINTER(_Matrix)
        L.nuq_create.argtypes = [ctypes.c_int, ctypes.c_char_p, ctypes.c_size_t]
        L.nuq_create.restype = vp
        L.nuq_destroy.argtypes = [vp]
        L.nuq_destroy.restype = None
        L.nuq_set_stream.argtypes = [vp, vp]
        L.nuq_reserve_workspace.argtypes = [vp, u64]
        L.nuq_workspace_bytes.argtypes = [vp]
        L.nuq_workspace_bytes.restype = u64
        L.nuq_sync.argtypes = [vp]
        L.nuq_last_error.argtypes = [vp]
        L.nuq_last_error.restype = ctypes.c_char_p
        L.nuq_set_generic_only.argtypes = [vp, ctypes.c_int]
        L.nuq_validate_row.argtypes = [u32, u64, u64]
        L.nuq_embed.argtypes = [vp, mp, u32, vp]
        L.nuq_dequant_range.argtypes = [vp, mp, u64, u64, vp]
        L.nuq_dequant_rows.argtypes = [vp, u32, vp, u64, u32, u32, vp]
        L.nuq_gemv.argtypes = [vp, u32, vp, u64, u32, u32, vp, vp]
        L.nuq_gemm.argtypes = [vp, u32, vp, u64, u32, u32, vp, u32, u64, vp, u64, u32]
        L.nuq_topk.argtypes = [vp, vp, u64, u32, ctypes.c_float, ctypes.POINTER(_TopKBuffers)]
        L.nuq_penalize.argtypes = [vp, vp, u64, vp, u64, ctypes.c_float, ctypes.c_float]
        L.nuq_matvec.argtypes = [vp, mp, vp, vp]
        L.nuq_matvec_rows.argtypes = [vp, mp, vp, u64, vp, u64, u32]
        L.nuq_matmul.argtypes = [vp, mp, vp, u32, u64, vp, u64, u32]
        L.nuq_matmul_kernel.argtypes = [vp, u32, mp, vp, u32, u64, vp, u64, u32]
        L.nuq_matvec_segments.argtypes = [vp, ctypes.POINTER(_Segment), u32, vp, u32]
        L.nuq_matvec_segments_noalloc.argtypes = [vp, ctypes.POINTER(_Segment), u32, vp, u32]
        L.nuq_argmax.argtypes = [vp, vp, u64, ctypes.POINTER(u32)]
        L.nuq_quantize_rows.argtypes = [u32, vp, u64, u64, vp, u64]
        cp = ctypes.POINTER(_Cache)
        L.nuq_cache_bytes.argtypes = [cp, ctypes.POINTER(u64)]
        L.nuq_cache_write.argtypes = [vp, cp, vp, vp, u32, u64, u64, vp, u64]
        L.nuq_cache_read.argtypes = [vp, cp, vp, u64, u32, vp, vp, u64, u64]
        L.nuq_cache_attention.argtypes = [vp, cp, ctypes.POINTER(_Attention)]
        L.nuq_logprobs.argtypes = [vp, vp, u32, u64, u64, u64, vp, u32, vp, vp, vp, vp]
        _lib = L
    return _lib


def _raise(code: int, message: str = "") -> None:
    if code != 0:
        cls = _ERRORS.get(code, NuqError)
        raise cls(message or cls.__name__)


def validate_row(encoding: int, byte_count: int, element_count: int) -> None:
    """decode.validateRow (quant/decode.zig:108-120)."""
    _raise(lib().nuq_validate_row(encoding, byte_count, element_count))


def row_bytes(encoding: int, columns: int) -> int:
    values, size = LAYOUT[encoding]
    return columns // values * size


def quantize(encoding: int, weights: np.ndarray) -> np.ndarray:
    """F32 [rows][columns] -> GGUF rows (uint8 [rows][row_bytes]) on the host.

    Q8_0 is the reference's q8_0Row (quant/encode.zig:17-36); Q4_K, Q5_K, Q6_K
    and IQ4_XS use this library's own quantizers (the reference has none)."""
    w = np.ascontiguousarray(weights, dtype=np.float32)
    if w.ndim == 1:
        w = w[None, :]
    rows, columns = w.shape
    if encoding not in LAYOUT:
        raise UnsupportedTensorEncoding("UnsupportedTensorEncoding")
    if columns % LAYOUT[encoding][0]:
        raise InvalidRowLength("InvalidRowLength")
    out = np.empty((rows, row_bytes(encoding, columns)), dtype=np.uint8)
    _raise(lib().nuq_quantize_rows(encoding, w.ctypes.data, rows, columns, out.ctypes.data, out.size))
    return out


@dataclass
class Matrix:
    """cpu.Matrix (backends/cpu/root.zig:31-36) whose bytes live on the GPU.

    `bytes` is a torch uint8 CUDA tensor (or anything with data_ptr/numel);
    `byte_len` defaults to its size."""

    encoding: int
    rows: int
    columns: int
    bytes: object
    byte_len: int | None = None

    def c(self) -> _Matrix:
        n = self.byte_len if self.byte_len is not None else self.bytes.numel() * self.bytes.element_size()
        return _Matrix(self.encoding, 0, self.rows, self.columns, self.bytes.data_ptr(), n)


def cache_bytes(bits: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int) -> int:
    """Device bytes of a KVCache of these sizes."""
    n = ctypes.c_uint64(0)
    for value in (bits, page_tokens, kv_heads, head_dim):
        if not 0 <= value < 1 << 32:
            raise InvalidShape(f"InvalidShape: {value}")
    _raise(lib().nuq_cache_bytes(ctypes.byref(_Cache(bits, page_tokens, kv_heads, head_dim, pages, None, 0)),
                                 ctypes.byref(n)))
    return n.value


class KVCache:
    """The quantised K/V cache of one layer (nuq_cache, include/nuq.h): `pages`
    pages of `page_tokens` tokens, 4 or 8 bits. Token t of page p is slot
    p * page_tokens + t. `bytes` is a contiguous uint8 CUDA tensor of
    cache_bytes(...) bytes; by default a new one of zeros."""

    def __init__(self, bits: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int, bytes=None, device=0):
        self.bits, self.pages, self.page_tokens = bits, pages, page_tokens
        self.kv_heads, self.head_dim = kv_heads, head_dim
        if bytes is None:
            import torch
            bytes = torch.zeros(cache_bytes(bits, pages, page_tokens, kv_heads, head_dim), dtype=torch.uint8,
                                device=f"cuda:{device}")
        elif not bytes.is_contiguous():
            raise InvalidShape("InvalidShape: the cache's bytes are not contiguous")
        self.bytes, self.device = bytes, bytes.get_device()
        self._ref = ctypes.byref(_Cache(bits, page_tokens, kv_heads, head_dim, pages, bytes.data_ptr(),
                                        bytes.numel() * bytes.element_size()))


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


class Backend:
    """One libnuq context on one GPU, launching on torch's current stream."""

    def __init__(self, device: int = 0):
        import torch

        self._torch = torch
        self.device = device
        self._float_codes = {torch.float32: F32, torch.float16: F16}
        # the current stream's handle without a Stream object around it (1 us a call)
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._raw_stream = raw or (lambda d: torch.cuda.current_stream(d).cuda_stream)
        err = ctypes.create_string_buffer(512)
        with torch.cuda.device(device):
            self._h = lib().nuq_create(device, err, len(err))
        if not self._h:
            raise DeviceError(err.value.decode())

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib().nuq_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- plumbing -----------------------------------------------------------
    def _call(self, fn, *args) -> None:
        stream = self._raw_stream(self.device)
        # a change of stream makes the new one wait for the old one's work
        # (the context's workspace is shared by its calls)
        code = lib().nuq_set_stream(self._h, stream)
        if code == 0:
            code = fn(self._h, *args)
        if code != 0:
            _raise(code, lib().nuq_last_error(self._h).decode())

    def sync(self) -> None:
        """nu_metal_commit's wait (bridge.m:279-310)."""
        self._call(lib().nuq_sync)

    def reserve_workspace(self, nbytes: int) -> None:
        """Allocates the device workspace up front (for graph capture)."""
        self._call(lib().nuq_reserve_workspace, nbytes)

    def workspace_bytes(self) -> int:
        return int(lib().nuq_workspace_bytes(self._h))

    def set_generic_only(self, enabled: bool) -> None:
        """Backend.generic_only (backends/metal/root.zig:99-102)."""
        lib().nuq_set_generic_only(self._h, int(enabled))

    # -- the reference's entry points ----------------------------------------
    def embed(self, matrix: Matrix, token: int, output) -> None:
        m = matrix.c()
        self._call(lib().nuq_embed, ctypes.byref(m), token, _ptr(output))

    def dequant_rows(self, matrix: Matrix, first: int, count: int, output) -> None:
        m = matrix.c()
        self._call(lib().nuq_dequant_range, ctypes.byref(m), first, count, _ptr(output))

    def matvec(self, matrix: Matrix, input, output) -> None:
        m = matrix.c()
        self._call(lib().nuq_matvec, ctypes.byref(m), _ptr(input), _ptr(output))

    def matvec_rows(self, matrix: Matrix, input, in_stride: int, output, out_stride: int, tokens: int) -> None:
        m = matrix.c()
        self._call(lib().nuq_matvec_rows, ctypes.byref(m), _ptr(input), in_stride, _ptr(output), out_stride, tokens)

    def matmul(self, matrix: Matrix, input, in_stride: int, output, out_stride: int, tokens: int) -> None:
        m = matrix.c()
        dtype = F16 if input.dtype == self._torch.float16 else F32
        self._call(lib().nuq_matmul, ctypes.byref(m), _ptr(input), dtype, in_stride, _ptr(output), out_stride, tokens)

    def matmul_kernel(self, kernel: int, matrix: Matrix, input, in_stride: int, output, out_stride: int,
                      tokens: int) -> None:
        m = matrix.c()
        dtype = F16 if input.dtype == self._torch.float16 else F32
        self._call(lib().nuq_matmul_kernel, kernel, ctypes.byref(m), _ptr(input), dtype, in_stride, _ptr(output),
                   out_stride, tokens)

    def matvec_segments(self, segments: list[tuple[Matrix, object]], input, mode: int = SEGMENT_PLAIN) -> None:
        arr = (_Segment * max(1, len(segments)))()
        for i, (mat, out) in enumerate(segments):
            arr[i].matrix = mat.c()
            arr[i].output = _ptr(out)
        self._call(lib().nuq_matvec_segments, arr, len(segments), _ptr(input), mode)

    def matvec_segments_noalloc(self, segments: list[tuple[Matrix, object]], input, mode: int = SEGMENT_PLAIN) -> None:
        """matvec_segments without any device allocation (no counterpart in
        the reference): the SiLU pair's second GEMV uses a fixed per-GPU
        scratch of NUQ_NOALLOC_MAX_PAIR_ROWS floats; calls that overlap on
        one GPU race on it."""
        arr = (_Segment * max(1, len(segments)))()
        for i, (mat, out) in enumerate(segments):
            arr[i].matrix = mat.c()
            arr[i].output = _ptr(out)
        self._call(lib().nuq_matvec_segments_noalloc, arr, len(segments), _ptr(input), mode)

    def penalize(self, logits, history_words, repetition: float, presence: float, count: int | None = None) -> None:
        """Backend.penalize (backends/metal/ops/sampling.zig:58-71), in place.
        `history_words` is a device uint32/int32 tensor: bit id of word id / 32."""
        n = logits.numel() if count is None else count
        self._call(lib().nuq_penalize, _ptr(logits), n, _ptr(history_words), history_words.numel(), repetition,
                   presence)

    def topk(self, logits, k: int, temperature: float, count: int | None = None) -> TopK:
        """Backend.topk (backends/metal/ops/sampling.zig:44-57) and the host's
        readback into sampling.TopK; synchronizes the stream."""
        torch = self._torch
        dev = logits.device
        values = torch.empty(max(k, 1), dtype=torch.float32, device=dev)
        indices = torch.empty(max(k, 1), dtype=torch.int32, device=dev)
        sums = torch.empty(TOPK_PARTIALS, dtype=torch.float32, device=dev)
        flags = torch.empty(TOPK_PARTIALS, dtype=torch.int32, device=dev)
        bufs = _TopKBuffers(values.data_ptr(), indices.data_ptr(), sums.data_ptr(), flags.data_ptr())
        n = logits.numel() if count is None else count
        self._call(lib().nuq_topk, _ptr(logits), n, k, temperature, ctypes.byref(bufs))
        self.sync()
        total = 0.0
        for partial in sums.cpu().tolist():  # F64, in partition order
            total += partial
        return TopK(temperature, [int(i) & 0xffffffff for i in indices.cpu().tolist()[:k]],
                    values.cpu().tolist()[:k], total, not bool(flags.cpu().any()))

    # -- the quantised cache and the attention over it ------------------------
    # (shapes, strides, dtypes and devices are asked for once each: a decode step
    # makes these calls for every layer, and each question to a tensor is 0.1 us;
    # an address of the host's would fault the GPU)
    def _elsewhere(self, t, name: str) -> InvalidArgument:
        return InvalidArgument(f"{name} is on {t.device}, not cuda:{self.device}")

    def _index(self, t, dtype, name: str):
        """The address of a contiguous tensor of this dtype on this device."""
        if t.get_device() != self.device:
            raise self._elsewhere(t, name)
        if t.dtype is not dtype:
            raise InvalidArgument(f"{name} must be {dtype}, not {t.dtype}")
        if not t.is_contiguous():
            raise InvalidShape(f"InvalidShape: {name} is not contiguous")
        return t.data_ptr()

    def _heads(self, t, head_dim: int, name: str):
        """Checks [rows][heads][head_dim] with contiguous rows on this device: (rows, heads, elements from a
        row to the next, the dtype's code)."""
        if t.get_device() != self.device:
            raise self._elsewhere(t, name)
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[2] != head_dim:
            raise InvalidShape(f"InvalidShape: {name} is {tuple(shape)}, not [rows][heads][{head_dim}]")
        rows, heads, _ = shape
        if stride[2] != 1 or (stride[1] != head_dim and heads > 1):
            raise InvalidShape(f"InvalidShape: {name}'s rows are not contiguous")
        code = self._float_codes.get(t.dtype)
        if code is None:
            raise InvalidArgument(f"{name} is {t.dtype}, not float32 or float16")
        return rows, heads, stride[0], code

    def _cache(self, cache: KVCache):
        if cache.device != self.device:
            raise self._elsewhere(cache.bytes, "the cache")
        return cache._ref

    def _slots(self, cache: KVCache, k, v, slots):
        tokens, heads, k_stride, code = self._heads(k, cache.head_dim, "k")
        v_tokens, v_heads, v_stride, v_code = self._heads(v, cache.head_dim, "v")
        if v_code != code:
            raise InvalidArgument("k and v differ in dtype")
        if heads != cache.kv_heads or v_heads != heads:
            raise InvalidShape(f"InvalidShape: {heads} and {v_heads} heads for a cache of {cache.kv_heads}")
        if slots.numel() != tokens or v_tokens != tokens:
            raise InvalidShape(f"InvalidShape: {slots.numel()} slots for {tokens} keys and {v_tokens} values")
        return code, tokens, k_stride, v_stride, self._index(slots, self._torch.int64, "slots")

    def cache_write(self, cache: KVCache, k, v, slots) -> None:
        """Quantises tokens' keys and values [tokens][kv_heads][head_dim] (F32
        or F16; rows may be strided) into their slots (int64; -1 skips)."""
        code, tokens, k_stride, v_stride, at = self._slots(cache, k, v, slots)
        self._call(_lib.nuq_cache_write, self._cache(cache), k.data_ptr(), v.data_ptr(), code, k_stride, v_stride, at, tokens)

    def cache_read(self, cache: KVCache, slots, k, v) -> None:
        """Reads slots back into k and v (F32 or F16, both exact)."""
        code, tokens, k_stride, v_stride, at = self._slots(cache, k, v, slots)
        self._call(_lib.nuq_cache_read, self._cache(cache), at, tokens, code, k.data_ptr(), v.data_ptr(), k_stride,
                   v_stride)

    def cache_attention(self, cache: KVCache, q, output, page_table, lengths, starts=None, scale: float | None = None,
                        window: int = 0, max_tokens: int | None = None, max_length: int = 0) -> None:
        """Causal attention of new tokens' queries [rows][q_heads][head_dim]
        over the cache (nuq_cache_attention, include/nuq.h). page_table int32
        [batch][pages], lengths int32 [batch] (the new tokens among them), starts
        int32 [batch + 1] where the sequences bring different counts of rows.
        `scale` is head_dim ** -0.5 by default; `max_tokens` (a bound on a
        sequence's rows) and `max_length` (on its tokens) size the launch."""
        rows, heads, q_stride, code = self._heads(q, cache.head_dim, "q")
        out_rows, out_heads, out_stride, out_code = self._heads(output, cache.head_dim, "output")
        if out_rows != rows or out_heads != heads or out_code != code:
            raise InvalidShape("InvalidShape: the output is not of q's shape and dtype")
        int32 = self._torch.int32
        batch = lengths.numel()
        table, table_stride = page_table.shape, page_table.stride()
        if len(table) != 2 or table[0] != batch:
            raise InvalidShape(f"InvalidShape: page table {tuple(table)} for {batch} sequences")
        if page_table.get_device() != self.device:
            raise self._elsewhere(page_table, "the page table")
        if page_table.dtype is not int32 or table_stride[1] != 1:
            raise InvalidArgument("the page table is not int32 with contiguous rows")
        first = None
        if starts is not None:
            if starts.numel() != batch + 1:
                raise InvalidShape(f"InvalidShape: {starts.numel()} starts for {batch} sequences")
            first = self._index(starts, int32, "starts")
        if max_tokens is None:
            max_tokens = rows if starts is not None else rows // max(batch, 1)
        if not (0 <= window < 1 << 32 and 0 <= max_tokens < 1 << 32 and 0 <= max_length < 1 << 63):
            raise InvalidShape(f"InvalidShape: window {window}, max_tokens {max_tokens}, max_length {max_length}")
        args = _Attention(q.data_ptr(), output.data_ptr(), code, heads, q_stride, out_stride, rows,
                          page_table.data_ptr(), table_stride[0], table[1], self._index(lengths, int32, "lengths"),
                          first, batch, max_tokens, max_length, cache.head_dim ** -0.5 if scale is None else scale,
                          window)
        self._call(_lib.nuq_cache_attention, self._cache(cache), ctypes.byref(args))

    def logprobs(self, logits, targets, logprobs, entropy, top_ids=None, top_logprobs=None) -> None:
        """Log probabilities of given tokens (nuq_logprobs, include/nuq.h):
        logits [rows][count] (F32 or F16, rows may be strided), targets int32
        [rows]; logprobs and entropy F32 [rows]; top_ids int32 and top_logprobs F32
        [rows][top], the most probable tokens (both or neither)."""
        torch = self._torch
        if logits.get_device() != self.device:
            raise self._elsewhere(logits, "the logits")
        shape, stride = logits.shape, logits.stride()
        if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
            raise InvalidShape(f"InvalidShape: logits {tuple(shape)} are not contiguous rows")
        code = self._float_codes.get(logits.dtype)
        if code is None:
            raise InvalidArgument(f"logits are {logits.dtype}, not float32 or float16")
        rows, count = shape
        if targets.numel() != rows or logprobs.numel() != rows or entropy.numel() != rows:
            raise InvalidShape(f"InvalidShape: targets or results are not of {rows} rows")
        if (top_ids is None) != (top_logprobs is None):
            raise InvalidArgument("top_ids and top_logprobs come together")
        top, ids, tops = 0, None, None
        if top_ids is not None:
            tops_shape = top_ids.shape
            if len(tops_shape) != 2 or tops_shape[0] != rows or tops_shape != top_logprobs.shape:
                raise InvalidShape(f"InvalidShape: top_ids {tuple(tops_shape)} and top_logprobs "
                                   f"{tuple(top_logprobs.shape)} for {rows} rows")
            top = tops_shape[1]
            ids = self._index(top_ids, torch.int32, "top_ids")
            tops = self._index(top_logprobs, torch.float32, "top_logprobs")
        self._call(_lib.nuq_logprobs, logits.data_ptr(), code, rows, count, stride[0],
                   self._index(targets, torch.int32, "targets"), top, self._index(logprobs, torch.float32, "logprobs"),
                   self._index(entropy, torch.float32, "entropy"), ids, tops)

    def argmax(self, logits) -> int:
        idx = ctypes.c_uint32(0)
        self._call(lib().nuq_argmax, _ptr(logits), logits.numel(), ctypes.byref(idx))
        return idx.value
