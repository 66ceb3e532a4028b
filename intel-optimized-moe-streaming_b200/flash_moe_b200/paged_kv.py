"""The paged key/value cache of the full-attention blocks and the attention
over it, on CUDA tensors (``include/moe_b200.h``, section 3).

Beside ``NativeDelta`` (the DeltaNet mixer's step) this is the other mixer of
the hybrid model: a serving loop writes each call's new keys and values and
attends over the cache, for prompts, chunks of prompts, drafted tokens and
single tokens alike::

    cache = PagedKVCache.empty(num_pages, page_size, kv_heads, head_dim, Q8_0, device)
    batch = KVBatch(q_start, kv_lens, page_table)   # int32 CUDA tensors
    cache.write(batch, k, v)                        # [tokens, kv_heads, head_dim]
    out = cache.attend(batch, q)                    # [tokens, q_heads, head_dim]
    k, v = cache.read(batch, dtype=torch.float16)   # the same rows, dequantised

Rows ``q_start[b] .. q_start[b+1]-1`` of the tokens belong to sequence b;
``kv_lens[b]`` counts its cached tokens, the new ones included.  All calls are
asynchronous on torch's current stream of the cache's device (or ``stream``),
read the batch on the device, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .formats import BF16, F16, F32, Q8_0

TYPE_IDS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
BLOCK_VALUES = 32   # values that share one scale of a Q8_0 cache


class KVBatch:
    """The sequences of a call: ``q_start`` [B + 1], ``kv_lens`` [B] and
    ``page_table`` [B, max_pages], int32 CUDA tensors.  Their contents may
    change between calls (a captured graph reads the current ones)."""

    def __init__(self, q_start: torch.Tensor, kv_lens: torch.Tensor, page_table: torch.Tensor):
        for t, dim in ((q_start, 1), (kv_lens, 1), (page_table, 2)):
            if t.dtype != torch.int32 or t.dim() != dim or not t.is_cuda:
                raise ValueError("KVBatch needs int32 CUDA tensors q_start [B + 1], kv_lens [B], "
                                 "page_table [B, max_pages]")
        n = kv_lens.shape[0]
        if q_start.shape[0] != n + 1 or page_table.shape[0] != n:
            raise ValueError("KVBatch shapes do not agree on the number of sequences")
        if not (q_start.device == kv_lens.device == page_table.device):
            raise ValueError("KVBatch tensors must be on one device")
        if not q_start.is_contiguous() or not kv_lens.is_contiguous() or (
                page_table.numel() and page_table.stride(1) != 1):
            raise ValueError("KVBatch tensors must have contiguous rows")
        if n > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ValueError("KVBatch page table rows must not overlap")
        self.q_start, self.kv_lens, self.page_table = q_start, kv_lens, page_table
        self.device = q_start.device
        self.sequences = n
        self.max_pages = page_table.shape[1]
        self._structs: dict[int, _lib.KVBatchStruct] = {}

    def struct(self, tokens: int) -> _lib.KVBatchStruct:
        s = self._structs.get(tokens)
        if s is None:
            if len(self._structs) > 64:
                self._structs.clear()
            stride = max(self.page_table.stride(0), self.max_pages)
            s = self._structs[tokens] = _lib.KVBatchStruct(
                self.sequences, tokens, self.max_pages, 0, stride, self.q_start.data_ptr(),
                self.kv_lens.data_ptr(), self.page_table.data_ptr())
        return s


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """Token and head strides of `t` [tokens, heads, dim]; 0 along an axis of
    one entry, whose stride torch leaves arbitrary."""
    ts, hs, _ = t.stride()
    return (ts if t.shape[0] > 1 else 0), (hs if t.shape[1] > 1 else 0)


def _aligned(t: torch.Tensor) -> bool:
    """Whether `t` [tokens, heads, dim] has contiguous, 16-byte aligned head
    rows."""
    step = 16 // t.element_size()
    ts, hs = _strides(t)
    return not (t.stride(2) != 1 or ts % step or hs % step or t.data_ptr() % 16)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t`, or a contiguous copy when its head rows are not aligned."""
    return t if _aligned(t) else t.clone(memory_format=torch.contiguous_format)


class PagedKVCache:
    """Keys and values [num_pages, kv_heads, page_size, head_dim]: fp16, bf16,
    or int8 codes with binary16 scales [..., head_dim / 32] (Q8_0 arithmetic:
    a value is scale * code).  The tensors are the caller's and are used in
    place."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor | None = None,
                 v_scales: torch.Tensor | None = None):
        self.lib = _lib.load()
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("cache k and v must be [num_pages, kv_heads, page_size, head_dim] "
                             "of one shape and dtype")
        pages, heads, page_size, dim = k.shape
        tensors = [k, v]
        if k.dtype == torch.int8:
            self.type = Q8_0
            shape = (pages, heads, page_size, dim // BLOCK_VALUES)
            for s in (k_scales, v_scales):
                if s is None or s.dtype != torch.float16 or tuple(s.shape) != shape:
                    raise ValueError(f"a Q8_0 cache needs fp16 scales of shape {shape}")
            tensors += [k_scales, v_scales]
        elif k.dtype in (torch.float16, torch.bfloat16):
            self.type = TYPE_IDS[k.dtype]
            if k_scales is not None or v_scales is not None:
                raise ValueError("only a Q8_0 cache has scales")
        else:
            raise ValueError("cache dtype must be fp16, bf16 or int8 (Q8_0)")
        if dim % BLOCK_VALUES or not 32 <= dim <= 256:
            raise ValueError("head_dim must be a multiple of 32 between 32 and 256")
        if page_size & (page_size - 1) or not 16 <= page_size <= 256:
            raise ValueError("page_size must be a power of two between 16 and 256")
        if pages < 1 or heads < 1 or heads > 1024 or pages * heads > 0x7fffffff:
            raise ValueError("the cache needs at least one page and 1 to 1024 heads, and fewer "
                             "than 2^31 pages * heads")
        for t in tensors:
            if not t.is_cuda or t.device != k.device or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("cache tensors must be contiguous, 16-byte aligned CUDA tensors "
                                 "on one device")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.device = k.device
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page_size, dim
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        self._struct = _lib.KVCacheStruct(self.type, pages, page_size, heads, dim, 0, ptr(k),
                                          ptr(v), ptr(k_scales), ptr(v_scales))
        self._ref = C.byref(self._struct)
        self._ws_bytes: dict[tuple, int] = {}

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, type_id: int,
              device) -> "PagedKVCache":
        """A cache of ``type_id`` F16, BF16 or Q8_0 (``formats``) with
        uninitialised pages."""
        dtype = {F16: torch.float16, BF16: torch.bfloat16, Q8_0: torch.int8}.get(type_id)
        if dtype is None:
            raise ValueError("cache type must be F16, BF16 or Q8_0")
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.int8:
            return cls(k, v)
        scales = (*shape[:3], head_dim // BLOCK_VALUES)
        return cls(k, v, *(torch.empty(scales, dtype=torch.float16, device=device)
                           for _ in range(2)))

    # ---------------------------------------------------------------- checks

    def _elsewhere(self, stream):
        """A context that makes `stream` current (and the cache's device), or
        None when the call can run as it is."""
        if stream is None:
            if torch.cuda.current_device() == self.device.index:
                return None
            return torch.cuda.device(self.device)
        if stream.device != self.device:
            raise ValueError("the stream must belong to the cache's device")
        return torch.cuda.stream(stream)

    def _check_rows(self, t, heads, dtypes, what):
        if (t.dim() != 3 or t.shape[1] != heads or t.shape[2] != self.head_dim
                or t.dtype not in dtypes or t.device != self.device):
            raise ValueError(f"{what} must be a [tokens, {heads}, {self.head_dim}] CUDA tensor on "
                             f"the cache's device, dtype one of {[str(d) for d in dtypes]}")

    def _check_output(self, t, what):
        if not _aligned(t):
            raise ValueError(f"{what} must have contiguous, 16-byte aligned head rows")

    def _status(self, status):
        if status is None:
            return None
        if status.dtype != torch.int32 or status.numel() < 1 or status.device != self.device:
            raise ValueError("status must be an int32 tensor on the cache's device")
        return status.data_ptr()

    # ----------------------------------------------------------------- calls

    def write(self, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, status=None,
              stream=None) -> None:
        """Store new rows k, v [tokens, kv_heads, head_dim] (fp32, fp16 or
        bf16, any strides) in the batch's pages (``moe_b200_kv_write``).
        ``status`` (int32 CUDA tensor, optional) receives 0 or a sum of
        ``_lib.KV_*`` bits."""
        other = self._elsewhere(stream)
        if other is not None:
            with other:
                return self.write(batch, k, v, status)
        self._check_rows(k, self.kv_heads, TYPE_IDS, "k")
        self._check_rows(v, self.kv_heads, (k.dtype,), "v")
        if k.shape != v.shape or batch.device != self.device:
            raise ValueError("k, v and the batch must agree in tokens and device")
        k, v = _rows(k), _rows(v)
        _lib.check(self.lib.moe_b200_kv_write(
            self._ref, batch.struct(k.shape[0]), TYPE_IDS[k.dtype], k.data_ptr(), *_strides(k),
            v.data_ptr(), *_strides(v), self._status(status),
            torch.cuda.current_stream(self.device).cuda_stream), "moe_b200_kv_write")

    def read(self, batch: KVBatch, tokens: int | None = None, dtype: torch.dtype | None = None,
             out: tuple[torch.Tensor, torch.Tensor] | None = None, status=None, stream=None):
        """The cached (k, v) at the batch's rows, [tokens, kv_heads, head_dim]
        of ``dtype`` (``moe_b200_kv_read``): with ``q_start`` the running sum
        of ``kv_lens``, whole sequences.  Give ``out``, or ``tokens`` and
        ``dtype`` (default: fp16 for a Q8_0 cache, else the cache's dtype);
        rows behind the last sequence are left as they are (uninitialised
        without ``out``)."""
        other = self._elsewhere(stream)
        if other is not None:
            with other:
                return self.read(batch, tokens, dtype, out, status)
        if out is None:
            if tokens is None or tokens < 0:
                raise ValueError("read needs out, or the number of tokens")
            if dtype is None:
                dtype = torch.float16 if self.type == Q8_0 else self.k.dtype
            shape = (tokens, self.kv_heads, self.head_dim)
            out = tuple(torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        k, v = out
        self._check_rows(k, self.kv_heads, TYPE_IDS, "out k")
        self._check_rows(v, self.kv_heads, (k.dtype,), "out v")
        if k.shape != v.shape or batch.device != self.device:
            raise ValueError("out and the batch must agree in tokens and device")
        self._check_output(k, "out k")
        self._check_output(v, "out v")
        _lib.check(self.lib.moe_b200_kv_read(
            self._ref, batch.struct(k.shape[0]), TYPE_IDS[k.dtype], k.data_ptr(), *_strides(k),
            v.data_ptr(), *_strides(v), self._status(status),
            torch.cuda.current_stream(self.device).cuda_stream), "moe_b200_kv_read")
        return k, v

    def attend(self, batch: KVBatch, q: torch.Tensor, out: torch.Tensor | None = None,
               lse: torch.Tensor | None = None, scale: float | None = None, causal: bool = True,
               window: int = 0, status=None, stream=None) -> torch.Tensor:
        """Attention of the batch's rows q [tokens, q_heads, head_dim] (fp16
        or bf16, the cache's own dtype unless it is Q8_0) over their cached
        tokens (``moe_b200_attend``).  ``scale`` defaults to
        head_dim ** -0.5; ``window`` > 0 keeps a causal row's last ``window``
        tokens; ``lse`` (fp32 [tokens, q_heads], contiguous) receives the
        logarithm of the softmax sum.  Rows without a token get zeros and
        -inf; rows behind the last sequence are left as they are (``out`` is
        allocated uninitialised when not given)."""
        other = self._elsewhere(stream)
        if other is not None:
            with other:
                return self.attend(batch, q, out, lse, scale, causal, window, status)
        dtypes = (torch.float16, torch.bfloat16) if self.type == Q8_0 else (self.k.dtype,)
        if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % self.kv_heads:
            raise ValueError("q must be [tokens, q_heads, head_dim], q_heads a multiple of "
                             "kv_heads")
        tokens, heads = q.shape[0], q.shape[1]
        self._check_rows(q, heads, dtypes, "q")
        if batch.device != self.device:
            raise ValueError("q and the batch must be on the cache's device")
        if window < 0 or (window and not causal):
            raise ValueError("window must be positive, and needs causal")
        q = _rows(q)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        else:
            self._check_rows(out, heads, (q.dtype,), "out")
            if out.shape[0] != tokens:
                raise ValueError("out must have q's shape")
            self._check_output(out, "out")
        if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (tokens, heads)
                                or not lse.is_contiguous() or lse.device != self.device):
            raise ValueError("lse must be a contiguous fp32 [tokens, q_heads] tensor on the "
                             "cache's device")
        bs = batch.struct(tokens)
        key = (tokens, heads, batch.sequences, batch.max_pages)
        need = self._ws_bytes.get(key)
        if need is None:
            n = C.c_size_t(0)
            _lib.check(self.lib.moe_b200_attend_workspace(self._ref, bs, heads, C.byref(n)),
                       "moe_b200_attend_workspace")
            if len(self._ws_bytes) > 4096:
                self._ws_bytes.clear()
            need = self._ws_bytes[key] = n.value
        # a workspace of the call's own: torch's allocator hands it to the next
        # call on this stream, or keeps it with the graph that captured it
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=self.device)
        _lib.check(self.lib.moe_b200_attend(
            self._ref, bs, TYPE_IDS[q.dtype], q.data_ptr(), *_strides(q), heads,
            out.data_ptr(), *_strides(out), lse.data_ptr() if lse is not None else None,
            self.head_dim ** -0.5 if scale is None else scale, 1 if causal else 0, window,
            ws.data_ptr(), ws.numel(), self._status(status),
            torch.cuda.current_stream(self.device).cuda_stream), "moe_b200_attend")
        return out
