"""Drafted decoding over a shared prompt: the quantised key/value cache, the
attention of a batch over one shared prefix, and the verification of drafts
(nb_kv_cache_* and nb_verify_drafts of include/needle_b200.h).

Tensors are torch tensors on the cache's GPU; work is queued on torch's current
stream of that GPU and nothing here waits for it, so the calls can be captured
into a CUDA graph.

    cache = nb.KvCache(kv_heads=4, head_dim=64, pages=1024, format="int8")
    batch = nb.KvBatch(row_start, lengths, pages, rows=R, max_rows=5, max_length=1000)
    cache.append(batch, keys, values)              # quantise the batch's new rows
    cache.attend(batch, query, out, prefix_pages, prefix_length)
    tokens, accepted = nb.verify_drafts(logits, draft_tokens, accept_uniforms, sample_uniforms, q)
"""

from __future__ import annotations

import ctypes
import math

from ._native import _check, lib

PAGE = 64
FORMATS = {"int8": 0, "e4m3": 1}
_DTYPES: dict = {}  # torch.dtype -> nb_dtype, filled with the first call
_torch = None


class nb_kv_batch(ctypes.Structure):
    _fields_ = [("sequences", ctypes.c_uint32), ("rows", ctypes.c_uint32), ("max_rows", ctypes.c_uint32), ("max_length", ctypes.c_uint32),
                ("page_stride", ctypes.c_uint32), ("row_start", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("pages", ctypes.c_void_p)]


class nb_rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class nb_verify(ctypes.Structure):
    _fields_ = [("sequences", ctypes.c_uint32), ("drafts", ctypes.c_uint32), ("vocab", ctypes.c_uint32), ("dtype", ctypes.c_int32),
                ("row_stride", ctypes.c_int64), ("logits", ctypes.c_void_p), ("draft_probabilities", ctypes.c_void_p),
                ("draft_tokens", ctypes.c_void_p), ("draft_counts", ctypes.c_void_p), ("mask_bits", ctypes.c_void_p),
                ("accept_uniforms", ctypes.c_void_p), ("sample_uniforms", ctypes.c_void_p), ("temperature", ctypes.c_float),
                ("tokens", ctypes.c_void_p), ("accepted", ctypes.c_void_p)]


_lib = None


def _library():
    global _lib, _torch
    L = lib()
    if _lib is not L:
        import torch

        _torch = torch
        _DTYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        P, U32, I32, SZ = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_size_t
        BATCH, ROWS = ctypes.POINTER(nb_kv_batch), ctypes.POINTER(nb_rows)
        sig = {
            "nb_kv_cache_create": (I32, [I32, I32, U32, U32, U32, ctypes.POINTER(P)]),
            "nb_kv_cache_release": (None, [P]),
            "nb_kv_cache_append": (I32, [P, BATCH, ROWS, ROWS, P]),
            "nb_kv_cache_read": (I32, [P, BATCH, ROWS, ROWS, P]),
            "nb_kv_cache_attend_workspace": (I32, [P, BATCH, U32, U32, ctypes.POINTER(SZ)]),
            "nb_kv_cache_attend": (I32, [P, BATCH, P, U32, ROWS, ROWS, U32, ctypes.c_float, P, SZ, P]),
            "nb_kv_cache_check": (I32, [P, P]),
            "nb_verify_drafts": (I32, [I32, ctypes.POINTER(nb_verify), P]),
        }
        for name, (res, args) in sig.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return L


def _stream(device: int) -> int:
    return _torch._C._cuda_getCurrentRawStream(device)


def _index_tensor(t, name: str, dims: int):
    """An int32 (or uint32) CUDA tensor, contiguous, of `dims` dimensions."""
    if not t.is_cuda or t.dim() != dims or not t.is_contiguous() or t.dtype not in (_torch.int32, getattr(_torch, "uint32", _torch.int32)):
        raise ValueError(f"{name} must be a contiguous int32 CUDA tensor of {dims} dimension(s)")
    return t


def _counts(**values) -> None:
    """Refuses what the C ABI's 32-bit counts do not hold; ctypes would drop the upper bits."""
    for name, value in values.items():
        if not 0 <= value < 1 << 32:
            raise ValueError(f"{name} must lie in [0, 2^32)")


class KvBatch:
    """The sequences of a call (nb_kv_batch): sequence b has the rows
    row_start[b] .. row_start[b + 1] of the dense tensors and lengths[b] cached
    positions, of which those rows are the last; its position p lies in page
    pages[b, p // 64]. The tensors are int32 on the cache's GPU and may be
    rewritten between calls; rows, max_rows and max_length bound them."""

    def __init__(self, row_start, lengths, pages, rows: int, max_rows: int, max_length: int):
        _library()
        _index_tensor(row_start, "row_start", 1)
        _index_tensor(lengths, "lengths", 1)
        _index_tensor(pages, "pages", 2)
        n = lengths.numel()
        if row_start.numel() != n + 1 or pages.shape[0] != n:
            raise ValueError("row_start holds one more entry than lengths, pages one row for each")
        if not row_start.device == lengths.device == pages.device:
            raise ValueError("row_start, lengths and pages must be on one GPU")
        _counts(rows=rows, max_rows=max_rows, max_length=max_length)
        self._kept = (row_start, lengths, pages)
        self.device = row_start.device.index
        self.rows = rows
        self._c = nb_kv_batch(n, rows, max_rows, max_length, pages.shape[1], row_start.data_ptr(), lengths.data_ptr(), pages.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._workspace: dict = {}  # (cache's heads and width, heads, prefix) -> bytes, all from the bounds above


class KvCache:
    """A pool of 64-position pages of 8-bit keys and values (nb_kv_cache_create):
    format "int8" (scale = peak * (1/127)) or "e4m3" (the smallest power of two)."""

    def __init__(self, kv_heads: int, head_dim: int, pages: int, format: str = "int8", device: int = -1):
        if format not in FORMATS:
            raise ValueError(f"format must be one of {sorted(FORMATS)}")
        _counts(kv_heads=kv_heads, head_dim=head_dim, pages=pages)
        L = _library()
        if device < 0 and _torch.cuda.is_available():
            device = _torch.cuda.current_device()
        h = ctypes.c_void_p()
        _check(L.nb_kv_cache_create(device, FORMATS[format], kv_heads, head_dim, pages, ctypes.byref(h)))
        self._h = h
        self.device, self.format, self.kv_heads, self.head_dim, self.pages = device, format, kv_heads, head_dim, pages

    def _rows(self, t, name: str, rows: int, heads: int) -> nb_rows:
        shape, stride = t.shape, t.stride()
        have = shape[0] if len(shape) == 3 else -1
        if have < rows or shape[1] != heads or shape[2] != self.head_dim or (stride[2] != 1 and have):
            raise ValueError(f"{name} must be [at least {rows} rows][{heads}][{self.head_dim}] with a contiguous last dimension")
        if t.get_device() != self.device or t.dtype not in _DTYPES:
            raise ValueError(f"{name} must be a float32, float16 or bfloat16 tensor on cuda:{self.device}")
        if not have:  # torch gives a tensor of no rows any strides
            stride = (heads * self.head_dim, self.head_dim)
        return nb_rows(t.data_ptr(), _DTYPES[t.dtype], stride[0], stride[1])

    def _batch(self, batch: KvBatch):
        if batch.device != self.device:
            raise ValueError(f"the batch is on cuda:{batch.device}, the cache on cuda:{self.device}")
        return batch._ref

    def append(self, batch: KvBatch, keys, values) -> None:
        """Quantises the batch's rows [rows][kv_heads][head_dim] into their positions."""
        k = self._rows(keys, "keys", batch.rows, self.kv_heads)
        v = self._rows(values, "values", batch.rows, self.kv_heads)
        _check(_lib.nb_kv_cache_append(self._h, self._batch(batch), k, v, _stream(self.device)))

    def read(self, batch: KvBatch, keys, values) -> None:
        """Reads the batch's rows back into keys and values, at the values they stand for."""
        k = self._rows(keys, "keys", batch.rows, self.kv_heads)
        v = self._rows(values, "values", batch.rows, self.kv_heads)
        _check(_lib.nb_kv_cache_read(self._h, self._batch(batch), k, v, _stream(self.device)))

    def attend(self, batch: KvBatch, query, out, prefix_pages=None, prefix_length: int = 0, scale: float | None = None) -> None:
        """Attention of the batch's rows over prefix_length shared positions and
        each sequence's own tail up to the row itself (nb_kv_cache_attend).
        query and out are [rows][heads][head_dim], float16 or bfloat16; scale
        defaults to 1 / sqrt(head_dim)."""
        heads = query.shape[1] if query.dim() == 3 else 0
        q = self._rows(query, "query", batch.rows, heads)
        o = self._rows(out, "out", batch.rows, heads)
        if not 0 <= prefix_length < 1 << 32:
            raise ValueError("prefix_length must lie in [0, 2^32)")
        pages = None
        if prefix_length:
            _index_tensor(prefix_pages, "prefix_pages", 1)
            if prefix_pages.numel() * PAGE < prefix_length or prefix_pages.get_device() != self.device:
                raise ValueError(f"prefix_pages must hold {-(-prefix_length // PAGE)} pages on cuda:{self.device}")
            pages = prefix_pages.data_ptr()
        ref = self._batch(batch)
        key = (self.kv_heads, self.head_dim, heads, prefix_length)
        size = batch._workspace.get(key)
        if size is None:
            n = ctypes.c_size_t()
            _check(_lib.nb_kv_cache_attend_workspace(self._h, ref, prefix_length, heads, ctypes.byref(n)))
            size = batch._workspace[key] = n.value
        # torch's allocator hands memory out stream by stream, and a captured graph keeps its own
        workspace = _torch.empty(size, dtype=_torch.uint8, device=query.device)
        _check(_lib.nb_kv_cache_attend(self._h, ref, pages, prefix_length, q, o, heads, 1.0 / math.sqrt(self.head_dim) if scale is None else scale,
                                       workspace.data_ptr(), size, _stream(self.device)))

    def check(self) -> None:
        """Waits for the current stream; raises if a call met a sequence out of
        its bounds or a page outside the pool since the last check."""
        _check(_lib.nb_kv_cache_check(self._h, _stream(self.device)))

    def close(self) -> None:
        if getattr(self, "_h", None):
            _lib.nb_kv_cache_release(self._h)
            self._h = None

    def __enter__(self) -> "KvCache":
        return self

    def __exit__(self, *exc) -> None:
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _plain(t, name: str, dtype, shape, device) -> int:
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on {device}")
    return t.data_ptr()


def verify_drafts(logits, draft_tokens, accept_uniforms, sample_uniforms, draft_probabilities=None, draft_counts=None, mask_bits=None,
                  temperature: float = 1.0, tokens=None, accepted=None):
    """Checks drafted tokens against the target's logits [n][drafts + 1][vocab]
    (nb_verify_drafts). draft_tokens [n][drafts] int32; accept_uniforms
    [n][drafts] and sample_uniforms [n] float32 in [0, 1) (None at temperature
    0); draft_probabilities [n][drafts][vocab] float32 or None (certain drafts);
    draft_counts [n] int32 or None; mask_bits [n][drafts + 1][ceil(vocab / 32)]
    int32 allowed ids or None. Returns (tokens [n][drafts + 1] int32, -1 behind
    the last; accepted [n] int32), written into the tensors given for them."""
    L = _lib or _library()
    torch = _torch
    if logits.dim() != 3 or (logits.stride(2) != 1 and logits.shape[0]) or logits.shape[1] < 1 or not logits.is_cuda or logits.dtype not in _DTYPES:
        raise ValueError("logits must be a float CUDA tensor [sequences][drafts + 1][vocab] with a contiguous last dimension")
    n, rows, vocab = logits.shape
    stride = vocab if n == 0 else logits.stride(1) if rows > 1 else logits.stride(0)
    if n > 1 and rows > 1 and logits.stride(0) != rows * stride:
        raise ValueError("the rows of logits must lie at one distance (a view of [sequences * (drafts + 1)] rows)")
    device, drafts = logits.device, rows - 1
    I32, F32 = torch.int32, torch.float32
    if tokens is None:
        tokens = torch.empty(n, rows, dtype=I32, device=device)
    if accepted is None:
        accepted = torch.empty(n, dtype=I32, device=device)
    if temperature != 0 and (accept_uniforms is None or sample_uniforms is None):
        raise ValueError("a temperature above 0 needs accept_uniforms and sample_uniforms")
    args = nb_verify(
        n, drafts, vocab, _DTYPES[logits.dtype], max(stride, vocab) if n * rows <= 1 else stride, logits.data_ptr(),
        None if draft_probabilities is None else _plain(draft_probabilities, "draft_probabilities", F32, (n, drafts, vocab), device),
        _plain(draft_tokens, "draft_tokens", I32, (n, drafts), device),
        None if draft_counts is None else _plain(draft_counts, "draft_counts", I32, (n,), device),
        None if mask_bits is None else _plain(mask_bits, "mask_bits", I32, (n, rows, (vocab + 31) // 32), device),
        None if accept_uniforms is None else _plain(accept_uniforms, "accept_uniforms", F32, (n, drafts), device),
        None if sample_uniforms is None else _plain(sample_uniforms, "sample_uniforms", F32, (n,), device),
        temperature, _plain(tokens, "tokens", I32, (n, rows), device), _plain(accepted, "accepted", I32, (n,), device))
    status = L.nb_verify_drafts(device.index, args, _stream(device.index))
    if status:
        _check(status)
    return tokens, accepted
